// The seam between two blocks of a residual network, forward and backward (sm_100a):
//   u = post(h);  y = x + f u, f = number * scale * gate;  z = norm(y)
// A CTA holds one row in registers at a time, a thread the same columns of every row, so that weights are fetched once
// and the column sums of the backward pass stay in registers until the CTA's rows are through.  Backward, with
//   t = dy + r (g - mean g - yn mean(g yn)),  g = dz * weight, yn = (y - mean) r   (rms: without mean g)
// dx = t, the branch's gradient is du = t f, and the inner norm takes du on to dh by the same formula.  y is made
// again from x and h, in 32 bits: its rounded copy would cost the weights' gradients their last digits.
// Sums over columns of the gradient go through one partial row per CTA, added up in a fixed order by a second kernel.
#include "training.h"

namespace ffcvb {

namespace {

using Args = ffcvb_norm_residual_args;

template <int V> struct Int { static constexpr int value = V; };

// N parameters from column `at` on, which is inside the row; `otherwise` without any.
template <int N>
__device__ __forceinline__ void load_params(float (&v)[N], const void *p, int type, int at, float otherwise) {
    if (!p) {
#pragma unroll
        for (int j = 0; j < N; j++) v[j] = otherwise;
    } else if constexpr (N == 1) {
        v[0] = type == FFCVB_TYPE_F32 ? static_cast<const float *>(p)[at]
               : type == FFCVB_TYPE_F16 ? to_float(static_cast<const __half *>(p)[at])
                                        : to_float(static_cast<const __nv_bfloat16 *>(p)[at]);
    } else if (type == FFCVB_TYPE_F32) {
#pragma unroll
        for (int j = 0; j < N; j += 4)
            *reinterpret_cast<float4 *>(v + j) = *reinterpret_cast<const float4 *>(static_cast<const float *>(p) + at + j);
    } else {
        uint32_t w[N / 2];
#pragma unroll
        for (int j = 0; j < N / 2; j += 2)
            *reinterpret_cast<uint2 *>(w + j) = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(p) + at + 2 * j);
#pragma unroll
        for (int j = 0; j < N / 2; j++) {
            const float2 two = type == FFCVB_TYPE_F16 ? __half22float2(*reinterpret_cast<const __half2 *>(w + j))
                                                      : make_float2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xffff0000u));
            v[2 * j] = two.x;
            v[2 * j + 1] = two.y;
        }
    }
}

// Sums over the threads of a row: a warp, a CTA, or (wide rows, backward) the CTAs of a cluster, whose sums travel through
// distributed shared memory.  Consecutive sums use `s` in turn, so that one barrier is enough.
template <bool MULTI> struct RowSum {
    float2 *s; // [2][32 + 4]
    int ctas = 1;
    int turn = 0;
    __device__ __forceinline__ float operator()(float a) { return (*this)(make_float2(a, 0.0f), false).x; }
    __device__ __forceinline__ float2 operator()(float2 v, bool both = true) {
        v.x = warp_sum(v.x);
        if (both) v.y = warp_sum(v.y);
        if constexpr (MULTI) {
            const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
            float2 *to = s + turn * 36;
            turn ^= 1;
            if (lane == 0) to[threadIdx.x >> 5] = v;
            __syncthreads();
            if (warps <= 8) {
                v = to[0];
                for (int k = 1; k < warps; k++) {
                    const float2 w = to[k];
                    v.x += w.x;
                    v.y += w.y;
                }
            } else {
                v = lane < warps ? to[lane] : make_float2(0.0f, 0.0f);
                v.x = warp_sum(v.x);
                if (both) v.y = warp_sum(v.y);
            }
            if (ctas > 1) {
                if ((int)threadIdx.x < ctas) {
                    uint32_t mine, rank, there;
                    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
                    mine = (uint32_t)__cvta_generic_to_shared(to + 32 + rank);
                    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(mine), "r"(threadIdx.x));
                    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(there), "f"(v.x), "f"(v.y) : "memory");
                }
                asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
                v = to[32];
                for (int k = 1; k < ctas; k++) {
                    const float2 w = to[32 + k];
                    v.x += w.x;
                    v.y += w.y;
                }
            }
        }
        return v;
    }
};

// A thread's columns: VPT packs of N, the packs of all threads of a row next to one another.
template <int N, int VPT, bool MULTI> struct Columns {
    int first, step, width;
    __device__ __forceinline__ Columns(long long w, int ctas = 1, int rank = 0) : width((int)w) {
        first = (MULTI ? rank * blockDim.x + threadIdx.x : threadIdx.x & 31) * N;
        step = (MULTI ? ctas * blockDim.x : 32) * N;
    }
    __device__ __forceinline__ int at(int k) const { return first + k * step; }
    __device__ __forceinline__ bool in(int k) const { return at(k) < width; } // (a pack is inside the row or not)
};

// Packs of coming rows on their way into shared memory, every thread's in places of its own, so that it waits for nobody
// else's.  Slots are used in turn.
__device__ __forceinline__ void copy16(void *to, const void *from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_made() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void copies_wait(int ahead) { // for the oldest of `ahead` (1 to 3) rows
    if (ahead == 3)
        asm volatile("cp.async.wait_group 2;" ::: "memory");
    else if (ahead == 2)
        asm volatile("cp.async.wait_group 1;" ::: "memory");
    else
        asm volatile("cp.async.wait_group 0;" ::: "memory");
}
// As many rows ahead, at most `most`, as shared memory has room for: it is shared by a CTA of 16 warps, or by CTAs of together as many.
constexpr size_t kRoom = 208 * 1024;
int rows_ahead(int most, size_t per_thread, size_t besides) {
    while (most > 1 && 512 * (most * per_thread + besides) > kRoom) most--;
    return most;
}

template <typename T, int N, int VPT, bool MULTI>
__device__ __forceinline__ void load_packs(Pack<T, N> (&v)[VPT], const void *p, long long offset, const Columns<N, VPT, MULTI> &c) {
#pragma unroll
    for (int k = 0; k < VPT; k++)
        if (c.in(k)) v[k].load(static_cast<const T *>(p) + offset + c.at(k));
}
// Values of packs, 0 beyond the row.
template <typename T, int N, int VPT, bool MULTI>
__device__ __forceinline__ void unpack(float (&v)[VPT][N], const Pack<T, N> (&p)[VPT], const Columns<N, VPT, MULTI> &c) {
#pragma unroll
    for (int k = 0; k < VPT; k++) {
        p[k].get(v[k]);
        if (!c.in(k)) {
#pragma unroll
            for (int j = 0; j < N; j++) v[k][j] = 0.0f;
        }
    }
}
template <typename T, int N, int VPT, bool MULTI>
__device__ __forceinline__ void load_row(float (&v)[VPT][N], const void *p, long long offset, const Columns<N, VPT, MULTI> &c) {
    Pack<T, N> raw[VPT];
    load_packs<T, N, VPT, MULTI>(raw, p, offset, c);
    unpack<T, N, VPT, MULTI>(v, raw, c);
}
template <typename T, int N, int VPT, bool MULTI>
__device__ __forceinline__ void store_row(const float (&v)[VPT][N], void *p, long long offset, const Columns<N, VPT, MULTI> &c) {
#pragma unroll
    for (int k = 0; k < VPT; k++)
        if (c.in(k)) {
            Pack<T, N> pack;
            pack.set(v[k]);
            pack.store(static_cast<T *>(p) + offset + c.at(k));
        }
}

// Mean (0 for rms) and 1 / deviation of a row: the mean first, then the squares of what is left.
template <int N, int VPT, bool MULTI>
__device__ __forceinline__ float2 row_stats(const float (&v)[VPT][N], int kind, const Columns<N, VPT, MULTI> &c, float eps, RowSum<MULTI> &sum) {
    const float over = 1.0f / (float)c.width;
    float mean = 0.0f;
    if (kind == FFCVB_NORM_LAYER) {
        float a = 0.0f;
#pragma unroll
        for (int k = 0; k < VPT; k++)
#pragma unroll
            for (int j = 0; j < N; j++) a += v[k][j];
        mean = sum(a) * over;
    }
    float q = 0.0f;
#pragma unroll
    for (int k = 0; k < VPT; k++)
        if (c.in(k)) {
#pragma unroll
            for (int j = 0; j < N; j++) q += (v[k][j] - mean) * (v[k][j] - mean);
        }
    return make_float2(mean, rsqrtf(sum(q) * over + eps));
}

// A row per warp, or (MULTI) per CTA.  Packs of more than one value need rows of a multiple of N values on 16-byte boundaries; the
// next rows of x and h (two, where there is room) are then on their way while one is worked on.
template <typename T, int N, int VPT, bool MULTI>
__global__ void __launch_bounds__(MULTI ? 512 : 128, MULTI ? 1 : 4)
forward_kernel(const __grid_constant__ Args a, const int ahead) {
    constexpr bool RING = N > 1;
    __shared__ float2 s_sum[72];
    extern __shared__ uint4 s_ring[]; // [ahead][2][VPT][threads]
    RowSum<MULTI> sum{s_sum};
    const Columns<N, VPT, MULTI> c(a.width);
    const long long step = MULTI ? gridDim.x : gridDim.x * 4ll;
    const long long begin = MULTI ? blockIdx.x : blockIdx.x * 4ll + (threadIdx.x >> 5);
    uint4 *const mine = s_ring + threadIdx.x;
    auto fetch = [&](long long row, int slot) {
        if (row < a.rows) {
#pragma unroll
            for (int k = 0; k < VPT; k++)
                if (c.in(k)) {
                    copy16(mine + (slot * 2 * VPT + k) * blockDim.x, static_cast<const T *>(a.x) + row * a.x_stride + c.at(k));
                    if (a.h) copy16(mine + (slot * 2 * VPT + VPT + k) * blockDim.x, static_cast<const T *>(a.h) + row * a.h_stride + c.at(k));
                }
        }
        copies_made();
    };
    if constexpr (RING)
        for (int k = 0; k < ahead; k++) fetch(begin + k * step, k);
    int slot = 0;
    for (long long row = begin; row < a.rows; row += step) {
        float y[VPT][N];
        float4 stats = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        Pack<T, N> raw[VPT], raw_h[VPT];
        if constexpr (RING) {
            copies_wait(ahead);
#pragma unroll
            for (int k = 0; k < VPT; k++)
                if (c.in(k)) {
                    raw[k].raw = mine[(slot * 2 * VPT + k) * blockDim.x];
                    if (a.h) raw_h[k].raw = mine[(slot * 2 * VPT + VPT + k) * blockDim.x];
                }
            fetch(row + ahead * step, slot);
            slot = slot + 1 == ahead ? 0 : slot + 1;
        } else {
            load_packs<T, N, VPT, MULTI>(raw, a.x, row * a.x_stride, c);
            if (a.h) load_packs<T, N, VPT, MULTI>(raw_h, a.h, row * a.h_stride, c);
        }
        if (a.h) {
            float u[VPT][N];
            unpack<T, N, VPT, MULTI>(u, raw_h, c);
            if (a.post_norm != FFCVB_NORM_NONE) {
                const float2 inner = row_stats<N, VPT, MULTI>(u, a.post_norm, c, a.eps, sum);
                stats.z = inner.x;
                stats.w = inner.y;
#pragma unroll
                for (int k = 0; k < VPT; k++)
                    if (c.in(k)) {
                        float w[N], b[N];
                        load_params<N>(w, a.post_weight, a.param_type, c.at(k), 1.0f);
                        load_params<N>(b, a.post_bias, a.param_type, c.at(k), 0.0f);
#pragma unroll
                        for (int j = 0; j < N; j++) u[k][j] = (u[k][j] - inner.x) * inner.y * w[j] + b[j];
                    }
            }
            if (a.gate_kind != FFCVB_GATE_NONE) {
                float gate[VPT][N];
                load_row<T, N, VPT, MULTI>(gate, a.gate, (a.gate_kind == FFCVB_GATE_SAMPLE ? row / a.tokens : row) * a.gate_stride, c);
#pragma unroll
                for (int k = 0; k < VPT; k++)
#pragma unroll
                    for (int j = 0; j < N; j++) u[k][j] *= gate[k][j];
            }
            unpack<T, N, VPT, MULTI>(y, raw, c);
#pragma unroll
            for (int k = 0; k < VPT; k++)
                if (c.in(k)) {
                    float f[N];
                    load_params<N>(f, a.scale, a.param_type, c.at(k), 1.0f);
#pragma unroll
                    for (int j = 0; j < N; j++) y[k][j] += u[k][j] * (a.number * f[j]);
                }
            store_row<T, N, VPT, MULTI>(y, a.y, row * a.width, c);
        } else {
            unpack<T, N, VPT, MULTI>(y, raw, c);
        }
        if (a.norm != FFCVB_NORM_NONE) {
            const float2 outer = row_stats<N, VPT, MULTI>(y, a.norm, c, a.eps, sum);
            stats.x = outer.x;
            stats.y = outer.y;
#pragma unroll
            for (int k = 0; k < VPT; k++)
                if (c.in(k)) {
                    float w[N], b[N];
                    load_params<N>(w, a.weight, a.param_type, c.at(k), 1.0f);
                    load_params<N>(b, a.bias, a.param_type, c.at(k), 0.0f);
#pragma unroll
                    for (int j = 0; j < N; j++) y[k][j] = (y[k][j] - outer.x) * outer.y * w[j] + b[j];
                }
            store_row<T, N, VPT, MULTI>(y, a.z, row * a.width, c);
        }
        if (a.stats && c.first == 0) reinterpret_cast<float4 *>(a.stats)[row] = stats;
    }
}

// How the backward pass deals its rows out.  A unit is a run of rows of one sample (with a gate per sample, whose
// gradient is a sum over them) or of all rows.
struct Deal {
    long long samples, tokens, splits, units;
    int threads, ctas_per_row, rows_at_once; // of a CTA; a cluster's CTAs; clusters
    int columns;                             // column sums of each cluster: weight, bias, post_weight, post_bias, scale
    int streams, ahead;                      // that are read; rows of them that are on their way (packs of 16 bytes)
};
// Partial rows: [rows_at_once][columns][width] of the column sums, then [units][width] of the gate's with more than one split.
struct Partials {
    float *columns, *gate;
};

constexpr int kColumns = 5;

template <int N, int VPT, bool MULTI>
__device__ __forceinline__ void store_floats(const float (&v)[VPT][N], float *to, const Columns<N, VPT, MULTI> &c) {
#pragma unroll
    for (int k = 0; k < VPT; k++)
        if (c.in(k)) {
#pragma unroll
            for (int j = 0; j < N; j++) to[c.at(k) + j] = v[k][j];
        }
}

// One row per CTA, or per cluster, at a time; with packs of 16 bytes those of the next are on their way meanwhile.
// POST: with an inner norm.  Of the branch's side two sums are kept per column and unit, A = sum t u and B = sum t (t with the gate,
// if it is one per token), u without weight and bias: all other gradients are made of them at a unit's end,
//   gate: f (pw A + pb B);  times the sample's gate:  scale: pw A + pb B,  post_weight: f A,  post_bias: f B.
template <typename T, int N, int VPT, bool MULTI, bool POST>
__global__ void __launch_bounds__(MULTI ? 512 : 32, MULTI ? 1 : 16)
backward_kernel(const __grid_constant__ Args a, const Deal deal, const Partials part) {
    constexpr bool RING = N > 1;
    __shared__ float2 s_sum[72];
    extern __shared__ uint4 s_ring[]; // [deal.ahead][deal.streams][VPT][threads], then floats [3][VPT * N][threads]: see below
    int rank = 0, cluster = blockIdx.x;
    if (MULTI && deal.ctas_per_row > 1) {
        rank = blockIdx.x % deal.ctas_per_row;
        cluster = blockIdx.x / deal.ctas_per_row;
    }
    RowSum<MULTI> sum{s_sum, deal.ctas_per_row};
    const Columns<N, VPT, MULTI> c(a.width, deal.ctas_per_row, rank);
    const float over = 1.0f / (float)a.width;
    const bool per_sample = a.gate_kind == FFCVB_GATE_SAMPLE;
    // with a gate per sample the sums over units are kept here, the thread's own
    float *const kept = reinterpret_cast<float *>(s_ring + (RING ? deal.ahead * deal.streams * VPT * blockDim.x : 0)) + threadIdx.x;
    if (per_sample)
        for (int k = 0; k < 3 * VPT * N; k++) kept[k * blockDim.x] = 0.0f;
    float dw[VPT][N] = {}, db[VPT][N] = {}, sa[VPT][N] = {}, sb[VPT][N] = {};
    float w[VPT][N], f[VPT][N];
#pragma unroll
    for (int k = 0; k < VPT; k++) {
        const int at = c.in(k) ? c.at(k) : 0;
        load_params<N>(w[k], a.weight, a.param_type, at, 1.0f);
        load_params<N>(f[k], a.scale, a.param_type, at, 1.0f);
#pragma unroll
        for (int j = 0; j < N; j++) f[k][j] *= a.number;
    }
    uint4 *const mine = s_ring + threadIdx.x;
    if (MULTI && deal.ctas_per_row > 1) // (all of a cluster's CTAs have begun before one writes into another's memory)
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    for (long long unit = cluster; unit < deal.units; unit += deal.rows_at_once) {
        const long long sample = unit / deal.splits, split = unit % deal.splits;
        const long long begin = sample * deal.tokens + deal.tokens * split / deal.splits;
        const long long end = sample * deal.tokens + deal.tokens * (split + 1) / deal.splits;
        float gate[VPT][N];
#pragma unroll
        for (int k = 0; k < VPT; k++)
#pragma unroll
            for (int j = 0; j < N; j++) gate[k][j] = 1.0f;
        if (per_sample) load_row<T, N, VPT, MULTI>(gate, a.gate, sample * a.gate_stride, c);
        auto fetch = [&](long long row, int slot) {
            if (row < end) {
                uint4 *to = mine + slot * deal.streams * VPT * blockDim.x;
                auto one = [&](const void *from, long long stride) {
                    if (!from) return;
#pragma unroll
                    for (int k = 0; k < VPT; k++)
                        if (c.in(k)) copy16(to + k * blockDim.x, static_cast<const T *>(from) + row * stride + c.at(k));
                    to += VPT * blockDim.x;
                };
                one(a.x, a.x_stride);
                one(a.h, a.h_stride);
                one(a.dy, a.dy_stride);
                one(a.dz, a.dz_stride);
                if (a.gate_kind == FFCVB_GATE_TOKEN) one(a.gate, a.gate_stride);
            }
            copies_made();
        };
        if constexpr (RING)
            for (int k = 0; k < deal.ahead; k++) fetch(begin + k, k);
        int slot = 0;
        for (long long row = begin; row < end; row++) {
            float y[VPT][N], u[VPT][N], t[VPT][N], dz[VPT][N];
            const float4 stats = reinterpret_cast<const float4 *>(a.stats)[row];
            if constexpr (RING) {
                copies_wait(deal.ahead);
                const uint4 *from = mine + slot * deal.streams * VPT * blockDim.x;
                auto one = [&](float(&v)[VPT][N], const void *there) {
                    Pack<T, N> raw[VPT] = {};
                    if (there) {
#pragma unroll
                        for (int k = 0; k < VPT; k++)
                            if (c.in(k)) raw[k].raw = from[k * blockDim.x];
                        from += VPT * blockDim.x;
                    }
#pragma unroll
                    for (int k = 0; k < VPT; k++) raw[k].get(v[k]);
                };
                one(y, a.x);
                one(u, a.h);
                one(t, a.dy);
                one(dz, a.dz);
                if (a.gate_kind == FFCVB_GATE_TOKEN) one(gate, a.gate);
                fetch(row + deal.ahead, slot);
                slot = slot + 1 == deal.ahead ? 0 : slot + 1;
            } else {
                auto one = [&](float(&v)[VPT][N], const void *from, long long stride) {
#pragma unroll
                    for (int k = 0; k < VPT; k++)
#pragma unroll
                        for (int j = 0; j < N; j++) v[k][j] = from && c.in(k) ? to_float(static_cast<const T *>(from)[row * stride + c.at(k) + j]) : 0.0f;
                };
                one(y, a.x, a.x_stride);
                one(u, a.h, a.h_stride);
                one(t, a.dy, a.dy_stride);
                one(dz, a.dz, a.dz_stride);
                if (a.gate_kind == FFCVB_GATE_TOKEN) one(gate, a.gate, a.gate_stride);
            }
            if (POST) { // u: normalised, without weight and bias
#pragma unroll
                for (int k = 0; k < VPT; k++)
#pragma unroll
                    for (int j = 0; j < N; j++) u[k][j] = (u[k][j] - stats.z) * stats.w;
            }
            // the inner norm's parameters are fetched again for every row, from L1: there are no registers for them
            auto post_params = [&](int k, float(&pw)[N], float(&pb)[N]) {
                load_params<N>(pw, a.post_weight, a.param_type, c.in(k) ? c.at(k) : 0, 1.0f);
                load_params<N>(pb, a.post_bias, a.param_type, c.in(k) ? c.at(k) : 0, 0.0f);
            };
            if (a.norm != FFCVB_NORM_NONE) {
                float2 means = make_float2(0.0f, 0.0f);
#pragma unroll
                for (int k = 0; k < VPT; k++) {
                    float pw[N], pb[N];
                    if (POST) post_params(k, pw, pb);
#pragma unroll
                    for (int j = 0; j < N; j++) {
                        const float whole = POST ? u[k][j] * pw[j] + pb[j] : u[k][j];
                        y[k][j] = (y[k][j] + whole * (f[k][j] * gate[k][j]) - stats.x) * stats.y;
                        dw[k][j] += dz[k][j] * y[k][j];
                        db[k][j] += dz[k][j];
                        dz[k][j] *= w[k][j];
                        means.x += dz[k][j];
                        means.y += dz[k][j] * y[k][j];
                    }
                }
                means = sum(means);
                const float m = a.norm == FFCVB_NORM_LAYER ? means.x * over : 0.0f, my = means.y * over;
#pragma unroll
                for (int k = 0; k < VPT; k++)
#pragma unroll
                    for (int j = 0; j < N; j++) t[k][j] = c.in(k) ? t[k][j] + stats.y * (dz[k][j] - m - y[k][j] * my) : 0.0f;
            }
            if (a.dx) store_row<T, N, VPT, MULTI>(t, a.dx, row * a.width, c);
            if (!a.h) continue;
            float2 means = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int k = 0; k < VPT; k++) {
                float pw[N], pb[N];
                if (POST) post_params(k, pw, pb);
#pragma unroll
                for (int j = 0; j < N; j++) {
                    if (a.gate_kind == FFCVB_GATE_TOKEN) { // (dz is not needed any more)
                        dz[k][j] = t[k][j] * (POST ? u[k][j] * pw[j] + pb[j] : u[k][j]) * f[k][j];
                        t[k][j] *= gate[k][j];
                    }
                    sa[k][j] += t[k][j] * u[k][j];
                    if (POST) sb[k][j] += t[k][j];
                    t[k][j] *= f[k][j];
                    if (per_sample) t[k][j] *= gate[k][j];
                    if (POST) {
                        t[k][j] *= pw[j];
                        means.x += t[k][j];
                        means.y += t[k][j] * u[k][j];
                    }
                }
            }
            if (a.gate_kind == FFCVB_GATE_TOKEN && a.dgate) store_row<T, N, VPT, MULTI>(dz, a.dgate, row * a.width, c);
            if (POST) {
                means = sum(means);
                const float m = a.post_norm == FFCVB_NORM_LAYER ? means.x * over : 0.0f, mu = means.y * over;
#pragma unroll
                for (int k = 0; k < VPT; k++)
#pragma unroll
                    for (int j = 0; j < N; j++) t[k][j] = stats.w * (t[k][j] - m - u[k][j] * mu);
            }
            if (a.dh) store_row<T, N, VPT, MULTI>(t, a.dh, row * a.width, c);
        }
        if (per_sample) {
            float dg[VPT][N];
#pragma unroll
            for (int k = 0; k < VPT; k++) {
                float pw[N], pb[N];
                load_params<N>(pw, a.post_weight, a.param_type, c.in(k) ? c.at(k) : 0, 1.0f);
                load_params<N>(pb, a.post_bias, a.param_type, c.in(k) ? c.at(k) : 0, 0.0f);
#pragma unroll
                for (int j = 0; j < N; j++) {
                    const float whole = pw[j] * sa[k][j] + pb[j] * sb[k][j];
                    float *to = kept + 3 * (k * N + j) * blockDim.x;
                    to[0] += f[k][j] * gate[k][j] * sa[k][j];
                    to[blockDim.x] += f[k][j] * gate[k][j] * sb[k][j];
                    to[2 * blockDim.x] += gate[k][j] * whole;
                    dg[k][j] = f[k][j] * whole;
                    sa[k][j] = sb[k][j] = 0.0f;
                }
            }
            if (a.dgate && deal.splits == 1)
                store_row<T, N, VPT, MULTI>(dg, a.dgate, sample * a.width, c);
            else if (a.dgate)
                store_floats<N, VPT, MULTI>(dg, part.gate + unit * a.width, c);
        }
    }
    float *to = part.columns + (long long)cluster * deal.columns * a.width;
    auto put = [&](const float(&v)[VPT][N], const void *wanted) {
        if (!wanted) return;
        store_floats<N, VPT, MULTI>(v, to, c);
        to += a.width;
    };
    put(dw, a.dweight);
    put(db, a.dbias);
#pragma unroll
    for (int k = 0; k < VPT; k++) {
        float pw[N], pb[N];
        load_params<N>(pw, a.post_weight, a.param_type, c.in(k) ? c.at(k) : 0, 1.0f);
        load_params<N>(pb, a.post_bias, a.param_type, c.in(k) ? c.at(k) : 0, 0.0f);
#pragma unroll
        for (int j = 0; j < N; j++) {
            const float *from = kept + 3 * (k * N + j) * blockDim.x;
            dw[k][j] = per_sample ? from[0] : f[k][j] * sa[k][j];
            db[k][j] = per_sample ? from[blockDim.x] : f[k][j] * sb[k][j];
            f[k][j] = a.number * (per_sample ? from[2 * blockDim.x] : pw[j] * sa[k][j] + pb[j] * sb[k][j]);
        }
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

// A thread of the backward pass has eight columns; up to 4096 of them are a CTA's, beyond that a cluster shares a row.
Deal deal_of(const Args &a) {
    Deal d{};
    d.ctas_per_row = (int)((a.width + 4095) / 4096);
    const int eights = (int)((a.width + 7) / 8);
    d.threads = ((eights + d.ctas_per_row - 1) / d.ctas_per_row + 31) / 32 * 32;
    const long long most = (long long)kSms * (512 / d.threads) / d.ctas_per_row; // 16 warps per SM
    d.samples = a.gate_kind == FFCVB_GATE_SAMPLE ? a.rows / a.tokens : 1;
    d.tokens = a.gate_kind == FFCVB_GATE_SAMPLE ? a.tokens : a.rows;
    if (d.samples < 1) d.samples = 1; // no rows
    // splits of a sample: those with which the longest turn of a cluster is shortest
    d.splits = 1;
    long long best = 0;
    const long long upto = d.samples >= most ? 8 : most / d.samples;
    for (long long s = d.samples >= most ? 1 : upto; s <= upto && s <= (d.tokens > 1 ? d.tokens : 1); s++) {
        const long long turn = (d.samples * s + most - 1) / most * ((d.tokens + s - 1) / s);
        if (!best || turn < best) {
            best = turn;
            d.splits = s;
        }
    }
    if (d.samples < most && d.splits == 1) d.splits = d.tokens < upto ? (d.tokens > 1 ? d.tokens : 1) : upto;
    d.units = d.samples * d.splits;
    d.rows_at_once = (int)(d.units < most ? d.units : most);
    for (const void *p : {a.dweight, a.dbias, a.dpost_weight, a.dpost_bias, a.dscale}) d.columns += p != nullptr;
    for (const void *p : {a.x, a.h, a.dy, a.dz, a.gate_kind == FFCVB_GATE_TOKEN ? a.gate : nullptr}) d.streams += p != nullptr;
    d.ahead = rows_ahead(3, d.streams * 8 * type_size(a.type), a.gate_kind == FFCVB_GATE_SAMPLE ? 96 : 0);
    return d;
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
    // up to 1024 values a warp has a row, then a CTA of a warp for every 1024; a lane has 8, 16, 24 or 32 of them
    const int warps = (int)((a.width + 1023) / 1024);
    const int eights = (int)((a.width + warps * 256 - 1) / (warps * 256));
    with_type(a.type, [&](auto zero) {
        using T = decltype(zero);
        constexpr int W = 16 / (int)sizeof(T);
        auto sized = [&](auto n) {
            constexpr int N = decltype(n)::value, V = 8 / N;
            auto run = [&](auto kernel, int per, long long ctas, int threads) {
                const int ahead = rows_ahead(2, 2 * per * V * 16, 0);
                const size_t room = N > 1 ? (size_t)ahead * 2 * per * V * threads * 16 : 0;
                if (room > 40 * 1024) cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)room);
                kernel<<<(unsigned)ctas, threads, room, st>>>(a, ahead);
            };
            if (warps == 1) {
                const long long all = (a.rows + 3) / 4, most = kSms * 16ll;
                run(eights == 1 ? forward_kernel<T, N, V, false> : eights == 2 ? forward_kernel<T, N, 2 * V, false>
                    : eights == 3 ? forward_kernel<T, N, 3 * V, false> : forward_kernel<T, N, 4 * V, false>, eights, all < most ? all : most, 128);
            } else {
                const long long most = kSms * (64ll / warps < 32 ? 64ll / warps : 32);
                run(eights <= 3 ? forward_kernel<T, N, 3 * V, true> : forward_kernel<T, N, 4 * V, true>, eights <= 3 ? 3 : 4, a.rows < most ? a.rows : most, 32 * warps);
            }
        };
        if (wide_rows(a))
            sized(Int<W>{});
        else
            sized(Int<1>{});
    });
    return launched("ffcvb_norm_residual");
}

int64_t ffcvb_norm_residual_workspace(const ffcvb_norm_residual_args *args) {
    if (!args || args->rows < 0 || args->width < 1 || (args->gate_kind == FFCVB_GATE_SAMPLE && args->tokens < 1)) return 0;
    const Deal d = deal_of(*args);
    return ((int64_t)d.rows_at_once * d.columns + (args->gate_kind == FFCVB_GATE_SAMPLE && d.splits > 1 ? d.units : 0)) * args->width * 4 + 16;
}

int ffcvb_norm_residual_backward(const ffcvb_norm_residual_args *args, void *stream) {
    if (const int rc = check(args, true)) return rc;
    const Args &a = *args;
    OnDevice here(a.device);
    if (!here.ok()) return training_fail(FFCVB_E_NODEVICE, "ffcvb_norm_residual_backward: no device %d", a.device);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const Deal d = deal_of(a);
    Partials part{static_cast<float *>(a.workspace), static_cast<float *>(a.workspace) + (long long)d.rows_at_once * d.columns * a.width};
    if (a.rows > 0)
        with_type(a.type, [&](auto zero) {
            using T = decltype(zero);
            auto sized = [&](auto n, auto post) {
                constexpr int N = decltype(n)::value, V = 8 / N;
                constexpr bool P = decltype(post)::value;
                const size_t room = (size_t)d.threads * V * ((N > 1 ? d.ahead * d.streams * 16 : 0) + (a.gate_kind == FFCVB_GATE_SAMPLE ? 12 * N : 0));
                auto run = [&](auto kernel) {
                    if (room > 40 * 1024) cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)room);
                    cudaLaunchConfig_t how{};
                    cudaLaunchAttribute cluster{};
                    cluster.id = cudaLaunchAttributeClusterDimension;
                    cluster.val.clusterDim.x = d.ctas_per_row;
                    cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
                    how.gridDim = dim3(d.rows_at_once * d.ctas_per_row);
                    how.blockDim = dim3(d.threads);
                    how.dynamicSmemBytes = room;
                    how.stream = st;
                    how.attrs = &cluster;
                    how.numAttrs = d.ctas_per_row > 1;
                    cudaLaunchKernelEx(&how, kernel, a, d, part);
                };
                run(d.threads == 32 && d.ctas_per_row == 1 ? backward_kernel<T, N, V, false, P> : backward_kernel<T, N, V, true, P>);
            };
            constexpr int W = 16 / (int)sizeof(T);
            const bool post = a.post_norm != FFCVB_NORM_NONE;
            if (wide_rows(a) && post)
                sized(Int<W>{}, Int<1>{});
            else if (wide_rows(a))
                sized(Int<W>{}, Int<0>{});
            else if (post)
                sized(Int<1>{}, Int<1>{});
            else
                sized(Int<1>{}, Int<0>{});
        });
    Sums s{};
    int n = 0;
    for (void *p : {a.dweight, a.dbias, a.dpost_weight, a.dpost_bias, a.dscale})
        if (p) {
            s.from[n] = part.columns + n * a.width;
            s.to[n++] = p;
        }
    s.width = a.width;
    s.count = a.rows > 0 ? d.rows_at_once : 0;
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
