// The seam between two blocks of a residual network, forward and backward (sm_100a):
//   u = post(h);  y = x + f u, f = number * scale * gate;  z = norm(y)
// A CTA holds one row in registers at a time, a thread the same columns of every row, so that weights are fetched once
// and the column sums of the backward pass stay in registers until the CTA's rows are through.  Backward, with
//   t = dy + r (g - mean g - yn mean(g yn)),  g = dz * weight, yn = (y - mean) r   (rms: without mean g)
// dx = t, the branch's gradient is du = t f, and the inner norm takes du on to dh by the same formula.  y is made
// again from x and h, in 32 bits: its rounded copy would cost the weights' gradients their last digits.
// Sums over columns of the gradient go through one partial row per CTA, added up in a fixed order by a second kernel.
#include "training.h"
#include "two.h"

namespace ffcvb {

namespace {

using Args = ffcvb_norm_residual_args;

template <int V> struct Int { static constexpr int value = V; };

// A thread's part of a row: eight columns, as 8 / N packs of N; the packs of all threads of a row lie next to one another.
// Arithmetic is on pairs of them.
constexpr int kPairs = 4;
using Eight = Two[kPairs];

template <int N, bool MULTI> struct Columns {
    int first, step, width;
    __device__ __forceinline__ Columns(long long w, int ctas, int rank) : width((int)w) {
        first = (MULTI ? rank * blockDim.x + threadIdx.x : threadIdx.x) * N;
        step = (MULTI ? ctas * blockDim.x : 32) * N;
    }
    __device__ __forceinline__ int at(int k) const { return first + k * step; }
    __device__ __forceinline__ bool in(int k) const { return at(k) < width; } // (a pack is inside the row or not)
};

__device__ __forceinline__ void fill(Eight &v, float value) {
#pragma unroll
    for (int p = 0; p < kPairs; p++) v[p] = Two(value, value);
}
template <typename T, int N>
__device__ __forceinline__ void to_pairs(Eight &v, const Pack<T, N> (&packs)[8 / N]) {
    float f[8];
#pragma unroll
    for (int k = 0; k < 8 / N; k++) packs[k].get(*reinterpret_cast<float(*)[N]>(f + k * N));
#pragma unroll
    for (int p = 0; p < kPairs; p++) v[p] = Two(f[2 * p], f[2 * p + 1]);
}
// Columns of a row in global memory; 0 beyond it.
template <typename T, int N, bool MULTI>
__device__ __forceinline__ void load_row(Eight &v, const void *p, long long offset, const Columns<N, MULTI> &c) {
    Pack<T, N> packs[8 / N] = {};
#pragma unroll
    for (int k = 0; k < 8 / N; k++)
        if (p && c.in(k)) packs[k].load(static_cast<const T *>(p) + offset + c.at(k));
    to_pairs<T, N>(v, packs);
}
template <typename T, int N, bool MULTI>
__device__ __forceinline__ void store_row(const Eight &v, void *p, long long offset, const Columns<N, MULTI> &c) {
    float f[8];
#pragma unroll
    for (int q = 0; q < kPairs; q++) {
        f[2 * q] = v[q].lo();
        f[2 * q + 1] = v[q].hi();
    }
#pragma unroll
    for (int k = 0; k < 8 / N; k++)
        if (c.in(k)) {
            Pack<T, N> pack;
            pack.set(*reinterpret_cast<const float(*)[N]>(f + k * N));
            pack.store(static_cast<T *>(p) + offset + c.at(k));
        }
}
// Parameters of the columns; `otherwise` without any, `beyond` beyond the row.
template <int N, bool MULTI>
__device__ __forceinline__ void load_params(Eight &v, const void *p, int type, const Columns<N, MULTI> &c, float otherwise, float beyond) {
    float f[8];
#pragma unroll
    for (int k = 0; k < 8 / N; k++) {
#pragma unroll
        for (int j = 0; j < N; j++) f[k * N + j] = c.in(k) ? otherwise : beyond;
        if (!p || !c.in(k)) continue;
        const int at = c.at(k);
        if constexpr (N == 1) {
            f[k] = type == FFCVB_TYPE_F32 ? static_cast<const float *>(p)[at]
                   : type == FFCVB_TYPE_F16 ? to_float(static_cast<const __half *>(p)[at])
                                            : to_float(static_cast<const __nv_bfloat16 *>(p)[at]);
        } else if (type == FFCVB_TYPE_F32) {
#pragma unroll
            for (int j = 0; j < N; j += 4) {
                const float4 w = *reinterpret_cast<const float4 *>(static_cast<const float *>(p) + at + j);
                f[k * N + j] = w.x, f[k * N + j + 1] = w.y, f[k * N + j + 2] = w.z, f[k * N + j + 3] = w.w;
            }
        } else {
#pragma unroll
            for (int j = 0; j < N; j += 4) {
                const uint2 w = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(p) + at + j);
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const uint32_t u = i ? w.y : w.x;
                    const float2 two = type == FFCVB_TYPE_F16 ? __half22float2(*reinterpret_cast<const __half2 *>(&u))
                                                              : make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
                    f[k * N + j + 2 * i] = two.x;
                    f[k * N + j + 2 * i + 1] = two.y;
                }
            }
        }
    }
#pragma unroll
    for (int q = 0; q < kPairs; q++) v[q] = Two(f[2 * q], f[2 * q + 1]);
}
template <int N, bool MULTI>
__device__ __forceinline__ void store_floats(const Eight &v, float *to, const Columns<N, MULTI> &c) {
#pragma unroll
    for (int k = 0; k < 8 / N; k++)
        if (c.in(k)) {
#pragma unroll
            for (int j = 0; j < N; j++) to[c.at(k) + j] = v[(k * N + j) / 2].half((k * N + j) & 1);
        }
}

// Two sums over the threads of a row: a warp, a CTA, or (wide rows) the CTAs of a cluster, whose sums travel through distributed
// shared memory.  In a warp the halves exchange what they do not go on with, so that two sums take little more than one.
// Consecutive sums use `s`, zero at the start, in turn, so that one barrier is enough.
template <bool MULTI> struct RowSum {
    float2 *s; // [2][32 + 4]
    int ctas;
    int turn = 0;
    __device__ __forceinline__ float2 operator()(float a, float b) {
        const int lane = threadIdx.x & 31;
        float v = lane & 16 ? b : a;
        v += __shfl_xor_sync(0xffffffffu, lane & 16 ? a : b, 16);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if constexpr (!MULTI) {
            return make_float2(__shfl_sync(0xffffffffu, v, 0), __shfl_sync(0xffffffffu, v, 16));
        } else {
            const int warps = blockDim.x >> 5;
            float2 *to = s + turn * 36;
            turn ^= 1;
            if ((lane & 15) == 0) reinterpret_cast<float *>(to + (threadIdx.x >> 5))[lane >> 4] = v;
            __syncthreads();
            float2 r = make_float2(0.0f, 0.0f);
            for (int k = 0; k < warps; k += 2) {
                const float4 w = *reinterpret_cast<const float4 *>(to + k);
                r.x += w.x + w.z;
                r.y += w.y + w.w;
            }
            if (ctas > 1) {
                if ((int)threadIdx.x < ctas) {
                    uint32_t mine, rank, there;
                    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
                    mine = (uint32_t)__cvta_generic_to_shared(to + 32 + rank);
                    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(mine), "r"(threadIdx.x));
                    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(there), "f"(r.x), "f"(r.y) : "memory");
                }
                cluster_barrier();
                r = to[32];
                for (int k = 1; k < ctas; k++) {
                    const float2 w = to[32 + k];
                    r.x += w.x;
                    r.y += w.y;
                }
            }
            return r;
        }
    }
    static __device__ __forceinline__ void cluster_barrier() {
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
    // (all of a cluster's CTAs have begun before one writes into another's memory)
    __device__ __forceinline__ void begin() {
        if constexpr (MULTI) {
            for (int k = threadIdx.x; k < 72; k += blockDim.x) s[k] = make_float2(0.0f, 0.0f);
            __syncthreads();
            if (ctas > 1) cluster_barrier();
        }
    }
};

__device__ __forceinline__ float sum_of(const Eight &v) {
    Two a = v[0];
#pragma unroll
    for (int p = 1; p < kPairs; p++) a = add_rn(a, v[p]);
    return a.lo() + a.hi();
}

// Packs of coming rows on their way into shared memory, every thread's in places of its own, so that it waits for nobody
// else's.  Slots are used in turn.
__device__ __forceinline__ void copy16(void *to, const void *from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_made() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void copies_wait(int ahead) { // for the oldest of `ahead` (1 to 3) rounds
    if (ahead == 3)
        asm volatile("cp.async.wait_group 2;" ::: "memory");
    else if (ahead == 2)
        asm volatile("cp.async.wait_group 1;" ::: "memory");
    else
        asm volatile("cp.async.wait_group 0;" ::: "memory");
}
// A thread's packs of one stream in a slot.
template <typename T, int N, bool MULTI>
__device__ __forceinline__ void copy_packs(uint4 *&to, const void *from, long long offset, const Columns<N, MULTI> &c) {
#pragma unroll
    for (int k = 0; k < 8 / N; k++)
        if (c.in(k)) copy16(to + k * blockDim.x, static_cast<const T *>(from) + offset + c.at(k));
    to += 8 / N * blockDim.x;
}
template <typename T, int N, bool MULTI>
__device__ __forceinline__ void copied(Eight &v, const uint4 *&from, const Columns<N, MULTI> &c) {
    Pack<T, N> packs[8 / N] = {};
#pragma unroll
    for (int k = 0; k < 8 / N; k++)
        if (c.in(k)) packs[k].raw = from[k * blockDim.x];
    to_pairs<T, N>(v, packs);
    from += 8 / N * blockDim.x;
}

// How rows are shared out: threads of a CTA, CTAs of a cluster, clusters; streams that are copied ahead and for how many rounds.
struct Shape {
    int threads, ctas_per_row, rows_at_once;
    int streams, ahead;
};

// Means and 1 / deviations of two rows: the means first (0 for rms), then the squares of what is left.
template <int N, bool MULTI>
__device__ __forceinline__ void two_stats(const Eight (&v)[2], int kind, const Columns<N, MULTI> &c, float eps, RowSum<MULTI> &sum, float (&mean)[2], float (&r)[2]) {
    const float over = 1.0f / (float)c.width;
    mean[0] = mean[1] = 0.0f;
    if (kind == FFCVB_NORM_LAYER) {
        const float2 both = sum(sum_of(v[0]), sum_of(v[1]));
        mean[0] = both.x * over;
        mean[1] = both.y * over;
    }
    float q[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const Two m(-mean[i], -mean[i]);
        Eight d;
#pragma unroll
        for (int p = 0; p < kPairs; p++) {
            d[p] = add_rn(v[i][p], m);
            d[p] = mul_rn(d[p], d[p]);
            if constexpr (N == 1)
                d[p] = Two(c.in(2 * p) ? d[p].lo() : 0.0f, c.in(2 * p + 1) ? d[p].hi() : 0.0f);
            else if (!c.in(2 * p / N))
                d[p] = Two(0.0f, 0.0f);
        }
        q[i] = sum_of(d);
    }
    const float2 both = sum(q[0], q[1]);
    r[0] = rsqrtf(both.x * over + eps);
    r[1] = rsqrtf(both.y * over + eps);
}
// (v - mean) r
__device__ __forceinline__ void normalise(Eight &v, float mean, float r) {
    const Two rr(r, r), m(-mean, -mean);
#pragma unroll
    for (int p = 0; p < kPairs; p++) v[p] = mul_rn(add_rn(v[p], m), rr);
}

// Two rows per CTA (or cluster, or warp) at a time, so that the sums of both take one barrier; with packs of 16 bytes those of the next
// rounds are on their way meanwhile.  POST: with an inner norm.
template <typename T, int N, bool MULTI, bool POST>
__global__ void __launch_bounds__(MULTI ? 512 : 32, MULTI ? 1 : 16)
forward_kernel(const __grid_constant__ Args a, const Shape shape) {
    constexpr bool RING = N > 1;
    __shared__ __align__(16) float2 s_sum[72];
    extern __shared__ uint4 s_ring[]; // [ahead][2][streams][8 / N][threads]
    int rank = 0, cluster = blockIdx.x;
    if (MULTI && shape.ctas_per_row > 1) {
        rank = blockIdx.x % shape.ctas_per_row;
        cluster = blockIdx.x / shape.ctas_per_row;
    }
    RowSum<MULTI> sum{s_sum, shape.ctas_per_row};
    sum.begin();
    const Columns<N, MULTI> c(a.width, shape.ctas_per_row, rank);
    Eight w, b, f, pw, pb; // (f is 0 beyond the row, which keeps y 0 there)
    load_params(w, a.weight, a.param_type, c, 1.0f, 1.0f);
    load_params(b, a.bias, a.param_type, c, 0.0f, 0.0f);
    load_params(f, a.scale, a.param_type, c, 1.0f, 0.0f);
    if (POST) {
        load_params(pw, a.post_weight, a.param_type, c, 1.0f, 1.0f);
        load_params(pb, a.post_bias, a.param_type, c, 0.0f, 0.0f);
    }
#pragma unroll
    for (int p = 0; p < kPairs; p++) f[p] = mul_rn(f[p], Two(a.number, a.number));
    const bool gated = a.gate_kind != FFCVB_GATE_NONE, per_sample = a.gate_kind == FFCVB_GATE_SAMPLE;
    const long long step = 2ll * shape.rows_at_once, begin = 2ll * cluster;
    // the sample of the next row to be fetched, and the row's place in it
    long long next_sample = per_sample ? begin / a.tokens : 0, next_place = per_sample ? begin % a.tokens : 0;
    const long long sample_step = per_sample ? step / a.tokens : 0, place_step = per_sample ? step % a.tokens : 0;
    uint4 *const mine = s_ring + threadIdx.x;
    const int slot_size = 2 * shape.streams * (8 / N) * blockDim.x;
    auto gate_row = [&](long long row, int i) { return per_sample ? next_sample + (i && next_place + 1 == a.tokens) : row + i; };
    auto fetched = [&]() {
        if (!per_sample) return;
        next_sample += sample_step;
        next_place += place_step;
        if (next_place >= a.tokens) {
            next_place -= a.tokens;
            next_sample++;
        }
    };
    auto fetch = [&](long long row, int slot) {
        uint4 *to = mine + slot * slot_size;
#pragma unroll
        for (int i = 0; i < 2; i++)
            if (row + i < a.rows) {
                copy_packs<T>(to, a.x, (row + i) * a.x_stride, c);
                if (a.h) copy_packs<T>(to, a.h, (row + i) * a.h_stride, c);
                if (gated) copy_packs<T>(to, a.gate, gate_row(row, i) * a.gate_stride, c);
            }
        copies_made();
        fetched();
    };
    if constexpr (RING)
        for (int k = 0; k < shape.ahead; k++) fetch(begin + k * step, k);
    int slot = 0;
    for (long long row = begin; row < a.rows; row += step) {
        const int rows = row + 1 < a.rows ? 2 : 1;
        Eight y[2], u[2], g[2];
        float4 stats[2] = {};
        if constexpr (RING) {
            copies_wait(shape.ahead);
            const uint4 *from = mine + slot * slot_size;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                if (i == 1 && rows == 1) from = mine + slot * slot_size; // (the same row again, to no effect)
                copied<T>(y[i], from, c);
                if (a.h) copied<T>(u[i], from, c);
                if (gated) copied<T>(g[i], from, c);
            }
            fetch(row + shape.ahead * step, slot);
            slot = slot + 1 == shape.ahead ? 0 : slot + 1;
        } else {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int k = i < rows ? i : 0;
                load_row<T>(y[i], a.x, (row + k) * a.x_stride, c);
                if (a.h) load_row<T>(u[i], a.h, (row + k) * a.h_stride, c);
                if (gated) load_row<T>(g[i], a.gate, gate_row(row, k) * a.gate_stride, c);
            }
            fetched();
        }
        if (a.h) {
            if (POST) {
                float mean[2], r[2];
                two_stats<N, MULTI>(u, a.post_norm, c, a.eps, sum, mean, r);
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    stats[i].z = mean[i];
                    stats[i].w = r[i];
                    normalise(u[i], mean[i], r[i]);
#pragma unroll
                    for (int p = 0; p < kPairs; p++) u[i][p] = fma_rn(u[i][p], pw[p], pb[p]);
                }
            }
#pragma unroll
            for (int i = 0; i < 2; i++) {
                if (gated)
#pragma unroll
                    for (int p = 0; p < kPairs; p++) u[i][p] = mul_rn(u[i][p], g[i][p]);
#pragma unroll
                for (int p = 0; p < kPairs; p++) y[i][p] = fma_rn(u[i][p], f[p], y[i][p]);
                if (i < rows) store_row<T>(y[i], a.y, (row + i) * a.width, c);
            }
        }
        if (a.norm != FFCVB_NORM_NONE) {
            float mean[2], r[2];
            two_stats<N, MULTI>(y, a.norm, c, a.eps, sum, mean, r);
#pragma unroll
            for (int i = 0; i < 2; i++) {
                stats[i].x = mean[i];
                stats[i].y = r[i];
                normalise(y[i], mean[i], r[i]);
#pragma unroll
                for (int p = 0; p < kPairs; p++) y[i][p] = fma_rn(y[i][p], w[p], b[p]);
                if (i < rows) store_row<T>(y[i], a.z, (row + i) * a.width, c);
            }
        }
        if (c.first == 0) {
            reinterpret_cast<float4 *>(a.stats)[row] = stats[0];
            if (rows == 2) reinterpret_cast<float4 *>(a.stats)[row + 1] = stats[1];
        }
    }
}

// How the backward pass deals its rows out.  A unit is a run of rows of one sample (with a gate per sample, whose
// gradient is a sum over them) or of all rows.
struct Deal {
    Shape shape;
    long long samples, tokens, splits, units;
    int columns; // column sums of each cluster: weight, bias, post_weight, post_bias, scale
};
// Partial rows: [rows_at_once][columns][width] of the column sums, then [units][width] of the gate's with more than one split.
struct Partials {
    float *columns, *gate;
};

constexpr int kColumns = 5;

// One row per CTA (or cluster, or warp) at a time; with packs of 16 bytes those of the next are on their way meanwhile.
// POST: with an inner norm.  Of the branch's side two sums are kept per column and unit, A = sum t u and B = sum t (t with the gate,
// if it is one per token), u without weight and bias: all other gradients are made of them at a unit's end,
//   gate: f (pw A + pb B);  times the sample's gate:  scale: pw A + pb B,  post_weight: f A,  post_bias: f B.
template <typename T, int N, bool MULTI, bool POST>
__global__ void __launch_bounds__(MULTI ? 512 : 32, MULTI ? 1 : 16)
backward_kernel(const __grid_constant__ Args a, const Deal deal, const Partials part) {
    constexpr bool RING = N > 1;
    const Shape &shape = deal.shape;
    __shared__ __align__(16) float2 s_sum[72];
    extern __shared__ uint4 s_ring[]; // [ahead][streams][8 / N][threads], then floats [8][3][threads]: see below
    int rank = 0, cluster = blockIdx.x;
    if (MULTI && shape.ctas_per_row > 1) {
        rank = blockIdx.x % shape.ctas_per_row;
        cluster = blockIdx.x / shape.ctas_per_row;
    }
    RowSum<MULTI> sum{s_sum, shape.ctas_per_row};
    sum.begin();
    const Columns<N, MULTI> c(a.width, shape.ctas_per_row, rank);
    const float over = 1.0f / (float)a.width;
    const bool per_sample = a.gate_kind == FFCVB_GATE_SAMPLE, per_token = a.gate_kind == FFCVB_GATE_TOKEN;
    const int slot_size = shape.streams * (8 / N) * blockDim.x;
    // with a gate per sample the sums over units are kept here, the thread's own
    float *const kept = reinterpret_cast<float *>(s_ring + (RING ? shape.ahead * slot_size : 0)) + threadIdx.x;
    if (per_sample)
        for (int k = 0; k < 24; k++) kept[k * blockDim.x] = 0.0f;
    Eight dw, db, sa, sb, w, f; // f: with the sample's gate; 0 beyond the row, which keeps everything of the branch 0 there
    fill(dw, 0.0f);
    fill(db, 0.0f);
    fill(sa, 0.0f);
    fill(sb, 0.0f);
    load_params(w, a.weight, a.param_type, c, 1.0f, 0.0f);
    auto load_f = [&]() {
        load_params(f, a.scale, a.param_type, c, 1.0f, 0.0f);
#pragma unroll
        for (int p = 0; p < kPairs; p++) f[p] = mul_rn(f[p], Two(a.number, a.number));
    };
    load_f();
    uint4 *const mine = s_ring + threadIdx.x;
    for (long long unit = cluster; unit < deal.units; unit += shape.rows_at_once) {
        const long long sample = unit / deal.splits, split = unit % deal.splits;
        const long long begin = sample * deal.tokens + deal.tokens * split / deal.splits;
        const long long end = sample * deal.tokens + deal.tokens * (split + 1) / deal.splits;
        if (per_sample) {
            Eight gate;
            load_f();
            load_row<T>(gate, a.gate, sample * a.gate_stride, c);
#pragma unroll
            for (int p = 0; p < kPairs; p++) f[p] = mul_rn(f[p], gate[p]);
        }
        auto fetch = [&](long long row, int slot) {
            if (row < end) {
                uint4 *to = mine + slot * slot_size;
                copy_packs<T>(to, a.x, row * a.x_stride, c);
                if (a.h) copy_packs<T>(to, a.h, row * a.h_stride, c);
                if (a.dy) copy_packs<T>(to, a.dy, row * a.dy_stride, c);
                if (a.dz) copy_packs<T>(to, a.dz, row * a.dz_stride, c);
                if (per_token) copy_packs<T>(to, a.gate, row * a.gate_stride, c);
            }
            copies_made();
        };
        if constexpr (RING)
            for (int k = 0; k < shape.ahead; k++) fetch(begin + k, k);
        float4 next = {};
        if (begin < end) next = reinterpret_cast<const float4 *>(a.stats)[begin];
        int slot = 0;
        for (long long row = begin; row < end; row++) {
            Eight y, u, t, dz, gate;
            const float4 stats = next;
            if (row + 1 < end) next = reinterpret_cast<const float4 *>(a.stats)[row + 1];
            fill(u, 0.0f);
            fill(t, 0.0f);
            fill(dz, 0.0f);
            if constexpr (RING) {
                copies_wait(shape.ahead);
                const uint4 *from = mine + slot * slot_size;
                copied<T>(y, from, c);
                if (a.h) copied<T>(u, from, c);
                if (a.dy) copied<T>(t, from, c);
                if (a.dz) copied<T>(dz, from, c);
                if (per_token) copied<T>(gate, from, c);
                fetch(row + shape.ahead, slot);
                slot = slot + 1 == shape.ahead ? 0 : slot + 1;
            } else {
                load_row<T>(y, a.x, row * a.x_stride, c);
                load_row<T>(u, a.h, row * a.h_stride, c);
                load_row<T>(t, a.dy, row * a.dy_stride, c);
                load_row<T>(dz, a.dz, row * a.dz_stride, c);
                if (per_token) load_row<T>(gate, a.gate, row * a.gate_stride, c);
            }
            Eight pw, pb; // fetched again for every row, from L1: there are no registers to keep them in
            if (POST) {
                normalise(u, stats.z, stats.w); // without weight and bias
                load_params(pw, a.post_weight, a.param_type, c, 1.0f, 1.0f);
                load_params(pb, a.post_bias, a.param_type, c, 0.0f, 0.0f);
            }
            if (a.norm != FFCVB_NORM_NONE) {
#pragma unroll
                for (int p = 0; p < kPairs; p++) {
                    const Two whole = POST ? fma_rn(u[p], pw[p], pb[p]) : u[p];
                    y[p] = fma_rn(per_token ? mul_rn(whole, gate[p]) : whole, f[p], y[p]);
                }
                normalise(y, stats.x, stats.y);
                Two first(0.0f, 0.0f), second(0.0f, 0.0f);
#pragma unroll
                for (int p = 0; p < kPairs; p++) {
                    dw[p] = fma_rn(dz[p], y[p], dw[p]);
                    db[p] = add_rn(db[p], dz[p]);
                    dz[p] = mul_rn(dz[p], w[p]);
                    first = add_rn(first, dz[p]);
                    second = fma_rn(dz[p], y[p], second);
                }
                const float2 means = sum(first.lo() + first.hi(), second.lo() + second.hi());
                const float m = a.norm == FFCVB_NORM_LAYER ? means.x * over : 0.0f, my = means.y * over;
                const Two minus_m(-m, -m), minus_my(-my, -my), r(stats.y, stats.y);
#pragma unroll
                for (int p = 0; p < kPairs; p++) t[p] = fma_rn(fma_rn(y[p], minus_my, add_rn(dz[p], minus_m)), r, t[p]);
            }
            if (a.dx) store_row<T>(t, a.dx, row * a.width, c);
            if (!a.h) continue;
            if (per_token) {
                Eight scale, dgate;
                load_params(scale, a.scale, a.param_type, c, 1.0f, 0.0f);
#pragma unroll
                for (int p = 0; p < kPairs; p++) {
                    const Two whole = POST ? fma_rn(u[p], pw[p], pb[p]) : u[p];
                    dgate[p] = mul_rn(mul_rn(t[p], whole), mul_rn(scale[p], Two(a.number, a.number)));
                    t[p] = mul_rn(t[p], gate[p]);
                }
                if (a.dgate) store_row<T>(dgate, a.dgate, row * a.width, c);
            }
            Two first(0.0f, 0.0f), second(0.0f, 0.0f);
#pragma unroll
            for (int p = 0; p < kPairs; p++) {
                sa[p] = fma_rn(t[p], u[p], sa[p]);
                if (POST) sb[p] = add_rn(sb[p], t[p]);
                t[p] = mul_rn(t[p], f[p]);
                if (POST) {
                    t[p] = mul_rn(t[p], pw[p]);
                    first = add_rn(first, t[p]);
                    second = fma_rn(t[p], u[p], second);
                }
            }
            if (POST) {
                const float2 means = sum(first.lo() + first.hi(), second.lo() + second.hi());
                const float m = a.post_norm == FFCVB_NORM_LAYER ? means.x * over : 0.0f, mu = means.y * over;
                const Two minus_m(-m, -m), minus_mu(-mu, -mu), r(stats.w, stats.w);
#pragma unroll
                for (int p = 0; p < kPairs; p++) t[p] = mul_rn(fma_rn(u[p], minus_mu, add_rn(t[p], minus_m)), r);
            }
            if (a.dh) store_row<T>(t, a.dh, row * a.width, c);
        }
        if (per_sample) {
            Eight dg, gate, pw, pb;
            load_params(pw, a.post_weight, a.param_type, c, 1.0f, 1.0f);
            load_params(pb, a.post_bias, a.param_type, c, 0.0f, 0.0f);
            load_row<T>(gate, a.gate, sample * a.gate_stride, c);
            load_f();
#pragma unroll
            for (int p = 0; p < kPairs; p++) {
                const Two whole = fma_rn(pw[p], sa[p], mul_rn(pb[p], sb[p])), fg = mul_rn(f[p], gate[p]);
                const Two add[3] = {mul_rn(fg, sa[p]), mul_rn(fg, sb[p]), mul_rn(gate[p], whole)};
#pragma unroll
                for (int j = 0; j < 6; j++) kept[(p * 6 + j) * blockDim.x] += add[j >> 1].half(j & 1);
                dg[p] = mul_rn(f[p], whole);
                sa[p] = sb[p] = Two(0.0f, 0.0f);
            }
            if (a.dgate && deal.splits == 1)
                store_row<T>(dg, a.dgate, sample * a.width, c);
            else if (a.dgate)
                store_floats(dg, part.gate + unit * a.width, c);
        }
    }
    float *to = part.columns + (long long)cluster * deal.columns * a.width;
    auto put = [&](const Eight &v, const void *wanted) {
        if (!wanted) return;
        store_floats(v, to, c);
        to += a.width;
    };
    put(dw, a.dweight);
    put(db, a.dbias);
    Eight pw, pb;
    load_params(pw, a.post_weight, a.param_type, c, 1.0f, 1.0f);
    load_params(pb, a.post_bias, a.param_type, c, 0.0f, 0.0f);
#pragma unroll
    for (int p = 0; p < kPairs; p++) {
        const float *from = kept + p * 6 * blockDim.x;
        const int next = blockDim.x;
        if (per_sample) {
            dw[p] = Two(from[0], from[next]);
            db[p] = Two(from[2 * next], from[3 * next]);
            f[p] = Two(from[4 * next], from[5 * next]);
        } else {
            dw[p] = mul_rn(f[p], sa[p]);
            db[p] = mul_rn(f[p], sb[p]);
            f[p] = fma_rn(pw[p], sa[p], mul_rn(pb[p], sb[p]));
        }
        f[p] = mul_rn(f[p], Two(a.number, a.number));
    }
    put(dw, a.dpost_weight);
    put(db, a.dpost_bias);
    put(f, a.dscale);
}

// Adds up partial rows: 32 columns per CTA, 32 runs of rows side by side.
struct Sums {
    const float *from[kColumns];
    void *to[kColumns];
    long long width, count, stride, from_z, to_z; // rows to add, from one to the next; from one sum (blockIdx.z) to the next
    int type;
};
__global__ void __launch_bounds__(1024)
add_up_kernel(const __grid_constant__ Sums s) {
    __shared__ float s_part[32][33];
    const int lane = threadIdx.x & 31, run = threadIdx.x >> 5;
    const long long c = blockIdx.x * 32ll + lane;
    const float *from = s.from[blockIdx.y] + blockIdx.z * s.from_z;
    float v = 0.0f;
    if (c < s.width) {
#pragma unroll 8
        for (long long r = run; r < s.count; r += 32) v += from[r * s.stride + c];
    }
    s_part[run][lane] = v;
    __syncthreads();
    v = warp_sum(s_part[lane][run]); // column `run`
    const long long mine = blockIdx.x * 32ll + run;
    if (lane == 0 && mine < s.width) {
        const long long at = blockIdx.z * s.to_z + mine;
        if (s.type == FFCVB_TYPE_F32)
            static_cast<float *>(s.to[blockIdx.y])[at] = v;
        else if (s.type == FFCVB_TYPE_F16)
            static_cast<__half *>(s.to[blockIdx.y])[at] = __float2half_rn(v);
        else
            static_cast<__nv_bfloat16 *>(s.to[blockIdx.y])[at] = __float2bfloat16_rn(v);
    }
}

bool wide_rows(const Args &a) {
    const int n = 16 / type_size(a.type);
    uintptr_t low = 0;
    for (const void *p : {a.x, a.h, a.gate, (const void *)a.y, (const void *)a.z, a.dy, a.dz, (const void *)a.dx, (const void *)a.dh, (const void *)a.dgate,
                          a.weight, a.bias, a.post_weight, a.post_bias, a.scale})
        low |= reinterpret_cast<uintptr_t>(p);
    return (low & 15) == 0 && (a.width | a.x_stride | (a.h ? a.h_stride : 0) | (a.gate ? a.gate_stride : 0) | (a.dy ? a.dy_stride : 0) |
                               (a.dz ? a.dz_stride : 0)) % n == 0;
}

// Rows of up to 4096 values are a CTA's (of up to 256 a warp's), wider ones a cluster's; as many rounds ahead, at most `most`, as shared
// memory has room for, which 16 warps per SM share.
constexpr size_t kRoom = 208 * 1024;
Shape shape_of(const Args &a, int streams, int most_ahead, size_t besides) {
    Shape s{};
    s.ctas_per_row = (int)((a.width + 4095) / 4096);
    const int eights = (int)((a.width + 7) / 8);
    s.threads = ((eights + s.ctas_per_row - 1) / s.ctas_per_row + 31) / 32 * 32;
    s.rows_at_once = kSms * (512 / s.threads) / s.ctas_per_row;
    s.streams = streams;
    s.ahead = most_ahead;
    while (s.ahead > 1 && 512 * ((size_t)s.ahead * streams * 8 * type_size(a.type) + besides) > kRoom) s.ahead--;
    return s;
}
Deal deal_of(const Args &a) {
    Deal d{};
    int streams = 0;
    for (const void *p : {a.x, a.h, a.dy, a.dz, a.gate_kind == FFCVB_GATE_TOKEN ? a.gate : nullptr}) streams += p != nullptr;
    d.shape = shape_of(a, streams, 3, a.gate_kind == FFCVB_GATE_SAMPLE ? 96 : 0);
    const long long most = d.shape.rows_at_once;
    d.samples = a.gate_kind == FFCVB_GATE_SAMPLE ? a.rows / a.tokens : 1;
    d.tokens = a.gate_kind == FFCVB_GATE_SAMPLE ? a.tokens : a.rows;
    if (d.samples < 1) d.samples = 1; // no rows
    // splits of a sample: those with which the longest turn of a cluster is shortest
    const long long least = d.samples >= most ? 1 : most / d.samples, upto = d.samples >= most ? 8 : least;
    long long best = 0;
    d.splits = 1;
    for (long long s = least; s <= upto; s++) {
        const long long splits = s < d.tokens ? s : d.tokens > 1 ? d.tokens : 1;
        const long long turn = (d.samples * splits + most - 1) / most * ((d.tokens + splits - 1) / splits);
        if (!best || turn < best) {
            best = turn;
            d.splits = splits;
        }
    }
    d.units = d.samples * d.splits;
    if (d.units < most) d.shape.rows_at_once = (int)d.units;
    for (const void *p : {a.dweight, a.dbias, a.dpost_weight, a.dpost_bias, a.dscale}) d.columns += p != nullptr;
    return d;
}

template <typename Kernel, typename... More>
void launch(Kernel kernel, const Shape &shape, size_t room, cudaStream_t stream, const More &...more) {
    // (what a CTA may have without being asked includes the static part)
    if (room > 40 * 1024) cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)room);
    cudaLaunchConfig_t how{};
    cudaLaunchAttribute cluster{};
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim.x = shape.ctas_per_row;
    cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
    how.gridDim = dim3(shape.rows_at_once * shape.ctas_per_row);
    how.blockDim = dim3(shape.threads);
    how.dynamicSmemBytes = room;
    how.stream = stream;
    how.attrs = &cluster;
    how.numAttrs = shape.ctas_per_row > 1;
    cudaLaunchKernelEx(&how, kernel, more...);
}

int check(const Args *args, bool backward) {
    const char *name = backward ? "ffcvb_norm_residual_backward" : "ffcvb_norm_residual";
    if (!args) return training_fail(FFCVB_E_ARG, "%s: no arguments", name);
    const Args &a = *args;
    auto type_ok = [](int t) { return t == FFCVB_TYPE_F32 || t == FFCVB_TYPE_F16 || t == FFCVB_TYPE_BF16; };
    auto norm_ok = [](int n) { return n >= FFCVB_NORM_NONE && n <= FFCVB_NORM_RMS; };
    if (a.width > FFCVB_NORM_MAX_WIDTH) return training_fail(FFCVB_E_LIMIT, "%s: rows of more than %d values", name, FFCVB_NORM_MAX_WIDTH);
    if (a.rows < 0 || a.width < 1 || !type_ok(a.type) || !type_ok(a.param_type) || !norm_ok(a.norm) || !norm_ok(a.post_norm) ||
        a.gate_kind < FFCVB_GATE_NONE || a.gate_kind > FFCVB_GATE_TOKEN)
        return training_fail(FFCVB_E_ARG, "%s: bad size, type or kind", name);
    if (a.rows > 0 && (!a.x || (a.gate_kind != FFCVB_GATE_NONE && !a.gate) || (!a.h && (a.post_norm != FFCVB_NORM_NONE || a.gate_kind != FFCVB_GATE_NONE || a.scale)) ||
                       (!a.h && a.norm == FFCVB_NORM_NONE)))
        return training_fail(FFCVB_E_ARG, "%s: bad argument", name);
    if ((a.gate_kind == FFCVB_GATE_SAMPLE && (a.tokens < 1 || a.rows % a.tokens)))
        return training_fail(FFCVB_E_ARG, "%s: bad argument", name);
    if (!backward && a.rows > 0 && ((a.norm != FFCVB_NORM_NONE && !a.z) || (a.h && !a.y)))
        return training_fail(FFCVB_E_ARG, "%s: no room for the results", name);
    if (backward && ((a.rows > 0 && !a.stats) || !a.workspace)) return training_fail(FFCVB_E_ARG, "%s: no statistics or workspace", name);
    return FFCVB_OK;
}

} // namespace

} // namespace ffcvb

using namespace ffcvb;

extern "C" {

int ffcvb_norm_residual(const ffcvb_norm_residual_args *args, void *stream) {
    if (const int rc = check(args, false)) return rc;
    const Args &a = *args;
    if (a.rows == 0) return FFCVB_OK;
    OnDevice here(a.device);
    if (!here.ok()) return training_fail(FFCVB_E_NODEVICE, "ffcvb_norm_residual: no device %d", a.device);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    Shape shape = shape_of(a, 1 + (a.h != nullptr) + (a.gate_kind != FFCVB_GATE_NONE), 2, 0);
    shape.streams *= 2; // (of two rows)
    while (shape.ahead > 1 && 512ull * shape.ahead * shape.streams * 8 * type_size(a.type) > kRoom) shape.ahead--;
    if ((a.rows + 1) / 2 < shape.rows_at_once) shape.rows_at_once = (int)((a.rows + 1) / 2);
    const bool wide = wide_rows(a), warp = shape.threads == 32 && shape.ctas_per_row == 1, post = a.post_norm != FFCVB_NORM_NONE;
    const size_t room = wide ? (size_t)shape.threads * shape.ahead * shape.streams * 8 * type_size(a.type) : 0;
    shape.streams /= 2;
    with_type(a.type, [&](auto zero) {
        using T = decltype(zero);
        auto sized = [&](auto n) {
            constexpr int N = decltype(n)::value;
            auto run = [&](auto kernel) { launch(kernel, shape, room, st, a, shape); };
            if (post)
                run(warp ? forward_kernel<T, N, false, true> : forward_kernel<T, N, true, true>);
            else
                run(warp ? forward_kernel<T, N, false, false> : forward_kernel<T, N, true, false>);
        };
        if (wide)
            sized(Int<16 / (int)sizeof(T)>{});
        else
            sized(Int<1>{});
    });
    return launched("ffcvb_norm_residual");
}

int64_t ffcvb_norm_residual_workspace(const ffcvb_norm_residual_args *args) {
    if (!args || args->rows < 0 || args->width < 1 || (args->gate_kind == FFCVB_GATE_SAMPLE && args->tokens < 1)) return 0;
    const Deal d = deal_of(*args);
    return ((int64_t)d.shape.rows_at_once * d.columns + (args->gate_kind == FFCVB_GATE_SAMPLE && d.splits > 1 ? d.units : 0)) * args->width * 4 + 16;
}

int ffcvb_norm_residual_backward(const ffcvb_norm_residual_args *args, void *stream) {
    if (const int rc = check(args, true)) return rc;
    const Args &a = *args;
    OnDevice here(a.device);
    if (!here.ok()) return training_fail(FFCVB_E_NODEVICE, "ffcvb_norm_residual_backward: no device %d", a.device);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const Deal d = deal_of(a);
    Partials part{static_cast<float *>(a.workspace), static_cast<float *>(a.workspace) + (long long)d.shape.rows_at_once * d.columns * a.width};
    if (a.rows > 0)
        with_type(a.type, [&](auto zero) {
            using T = decltype(zero);
            const Shape &shape = d.shape;
            const bool wide = wide_rows(a), warp = shape.threads == 32 && shape.ctas_per_row == 1, post = a.post_norm != FFCVB_NORM_NONE;
            const size_t room = (size_t)shape.threads * ((wide ? shape.ahead * shape.streams * 8 * sizeof(T) : 0) + (a.gate_kind == FFCVB_GATE_SAMPLE ? 96 : 0));
            auto sized = [&](auto n) {
                constexpr int N = decltype(n)::value;
                auto run = [&](auto kernel) { launch(kernel, shape, room, st, a, d, part); };
                if (post)
                    run(warp ? backward_kernel<T, N, false, true> : backward_kernel<T, N, true, true>);
                else
                    run(warp ? backward_kernel<T, N, false, false> : backward_kernel<T, N, true, false>);
            };
            if (wide)
                sized(Int<16 / (int)sizeof(T)>{});
            else
                sized(Int<1>{});
        });
    Sums s{};
    int n = 0;
    for (void *p : {a.dweight, a.dbias, a.dpost_weight, a.dpost_bias, a.dscale})
        if (p) {
            s.from[n] = part.columns + n * a.width;
            s.to[n++] = p;
        }
    s.width = a.width;
    s.count = a.rows > 0 ? d.shape.rows_at_once : 0;
    s.stride = d.columns * a.width;
    s.type = a.param_type;
    const unsigned across = (unsigned)((a.width + 31) / 32);
    if (n) add_up_kernel<<<dim3(across, n), 1024, 0, st>>>(s);
    if (a.dgate && a.gate_kind == FFCVB_GATE_SAMPLE && d.splits > 1 && a.rows > 0) {
        Sums g{};
        g.from[0] = part.gate;
        g.to[0] = a.dgate;
        g.width = g.stride = g.to_z = a.width;
        g.count = d.splits;
        g.from_z = d.splits * a.width;
        g.type = a.type;
        // (more than one split means that there are fewer samples than CTAs)
        add_up_kernel<<<dim3(across, 1, (unsigned)d.samples), 1024, 0, st>>>(g);
    }
    return launched("ffcvb_norm_residual_backward");
}

} // extern "C"
