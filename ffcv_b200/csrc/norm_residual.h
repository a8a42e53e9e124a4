// The seam between two blocks of a residual network: what its kernels share (sm_100a).
#pragma once

#include "training.h"
#include "two.h"

namespace ffcvb {

namespace norms {

using Args = ffcvb_norm_residual_args;

template <int V> struct Int { static constexpr int value = V; };

// A thread's part of a row: eight columns, as 8 / N packs of N, the packs of all threads of a row next to one another; single values are
// 32 apart (or as many as lanes have the row), and 256 next to one another a warp's.  Arithmetic is on pairs of them.  A row is a CTA's, a cluster's (CTA by CTA), or that
// of 8, 16 or 32 lanes of a CTA of one warp.
constexpr int kPairs = 4;
using Eight = Two[kPairs];

// LANES: 8, 16 or 32 of a CTA of one warp have a row; 0: all threads of a CTA or cluster.
template <int N, int LANES> struct Columns {
    static constexpr bool MULTI = LANES == 0;
    int thread, threads; // of the row, or of the CTA's part
    int part;            // first column of that
    int first, step, width;
    __device__ __forceinline__ Columns(long long w, int rank) : width((int)w) {
        thread = MULTI ? threadIdx.x : threadIdx.x & (LANES - 1);
        threads = MULTI ? blockDim.x : LANES;
        part = MULTI ? rank * blockDim.x * 8 : 0;
        first = part + (N == 1 ? (thread >> 5) * 256 + (thread & 31) : thread * N);
        step = N == 1 ? kApart : threads * N;
    }
    static constexpr int kApart = MULTI ? 32 : LANES; // of single values
    __device__ __forceinline__ int at(int k) const { return first + k * (N == 1 ? kApart : step); }
    __device__ __forceinline__ bool in(int k) const { return at(k) < width; } // (a pack is inside the row or not)
    __device__ __forceinline__ int inside(int k) const { return in(k) ? at(k) : 0; }
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
template <typename T, int N, int LANES>
__device__ __forceinline__ void load_row(Eight &v, const void *p, long long offset, const Columns<N, LANES> &c) {
    Pack<T, N> packs[8 / N] = {};
#pragma unroll
    for (int k = 0; k < 8 / N; k++)
        if (p && c.in(k)) packs[k].load(static_cast<const T *>(p) + offset + c.at(k));
    to_pairs<T, N>(v, packs);
}
template <typename T, int N, int LANES>
__device__ __forceinline__ void store_row(const Eight &v, void *p, long long offset, const Columns<N, LANES> &c) {
    float f[8];
#pragma unroll
    for (int q = 0; q < kPairs; q++) {
        f[2 * q] = v[q].lo();
        f[2 * q + 1] = v[q].hi();
    }
    T *const to = static_cast<T *>(p) + offset + c.first;
#pragma unroll
    for (int k = 0; k < 8 / N; k++)
        if (c.in(k)) {
            Pack<T, N> pack;
            pack.set(*reinterpret_cast<const float(*)[N]>(f + k * N));
            pack.store(to + k * (N == 1 ? c.kApart : c.step));
        }
}
// Parameters of the columns; `otherwise` without any, `beyond` beyond the row.
template <int N, int LANES>
__device__ __forceinline__ void load_params(Eight &v, const void *p, int type, const Columns<N, LANES> &c, float otherwise, float beyond) {
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
template <int N, int LANES>
__device__ __forceinline__ void store_floats(const Eight &v, float *to, const Columns<N, LANES> &c) {
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
template <int LANES> struct RowSum {
    static constexpr bool MULTI = LANES == 0;
    float2 *s; // [2][32 + 4]
    int ctas;
    int turn = 0;
    // the lanes of the thread's row
    __device__ __forceinline__ uint32_t mask() const { return MULTI || LANES == 32 ? 0xffffffffu : ((1u << (LANES & 31)) - 1) << (threadIdx.x & 31 & -LANES); }
    __device__ __forceinline__ float2 operator()(float a, float b) {
        const int lane = threadIdx.x & 31;
        if constexpr (!MULTI) {
            const uint32_t all = mask();
            constexpr int half = LANES / 2;
            float v = lane & half ? b : a;
            v += __shfl_xor_sync(all, lane & half ? a : b, half);
#pragma unroll
            for (int o = half / 2; o > 0; o >>= 1) v += __shfl_xor_sync(all, v, o);
            return make_float2(__shfl_sync(all, v, lane & -LANES), __shfl_sync(all, v, (lane & -LANES) + half));
        } else {
            float v = lane & 16 ? b : a;
            v += __shfl_xor_sync(0xffffffffu, lane & 16 ? a : b, 16);
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
            const int warps = blockDim.x >> 5;
            float2 *to = s + turn * 36;
            turn ^= 1;
            if ((lane & 15) == 0) reinterpret_cast<float *>(to + (threadIdx.x >> 5))[lane >> 4] = v;
            __syncthreads();
            float2 r;
            {
                const float4 w = *reinterpret_cast<const float4 *>(to), x = *reinterpret_cast<const float4 *>(to + 2);
                r = make_float2((w.x + w.z) + (x.x + x.z), (w.y + w.w) + (x.y + x.w)); // (0 without a warp)
            }
            for (int k = 4; k < warps; k += 2) {
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
// else's; zeros beyond the row.  Slots are used in turn.
__device__ __forceinline__ void copy16(uint32_t to, const void *from, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
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
// A thread's packs of one stream of a row that begins at `from`; `to` goes on to the next stream's places.
template <typename T, int N, int LANES>
__device__ __forceinline__ void copy_packs(uint32_t &to, const T *from, const Columns<N, LANES> &c) {
#pragma unroll
    for (int k = 0; k < 8 / N; k++) {
        copy16(to, from + c.inside(k), c.in(k) ? 16 : 0);
        to += blockDim.x * 16;
    }
}
template <typename T, int N>
__device__ __forceinline__ void copied(Eight &v, uint32_t &from) {
    Pack<T, N> packs[8 / N];
#pragma unroll
    for (int k = 0; k < 8 / N; k++) {
        uint4 &r = packs[k].raw;
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(from) : "memory");
        from += blockDim.x * 16;
    }
    to_pairs<T, N>(v, packs);
}

// Rows that do not begin on 16-byte boundaries: the packs that a row's part lies in are copied by its threads together, and its values
// read one by one from wherever they lie then.  A barrier of the row's threads is needed in between.
template <typename T> __host__ __device__ constexpr int window_bytes(int threads) { return threads * 8 * (int)sizeof(T) + 16; }
template <typename T, int LANES>
__device__ __forceinline__ void copy_window(uint32_t to, const T *row, const Columns<1, LANES> &c) {
    const T *from = row + c.part;
    const int lead = (int)(reinterpret_cast<uintptr_t>(from) & 15), bytes = lead + min(c.width - c.part, c.threads * 8) * (int)sizeof(T);
    const char *at = reinterpret_cast<const char *>(from) - lead;
    for (int k = c.thread * 16; k < bytes; k += c.threads * 16) copy16(to + k, at + k, 16);
}
template <typename T, int LANES>
__device__ __forceinline__ void window(Eight &v, uint32_t from, const T *row, const Columns<1, LANES> &c) {
    from += (uint32_t)(reinterpret_cast<uintptr_t>(row + c.part) & 15);
    const T *at = static_cast<const T *>(__cvta_shared_to_generic(from)) + (c.first - c.part);
    float f[8];
#pragma unroll
    for (int k = 0; k < 8; k++) f[k] = c.in(k) ? to_float(at[k * Columns<1, LANES>::kApart]) : 0.0f;
#pragma unroll
    for (int p = 0; p < kPairs; p++) v[p] = Two(f[2 * p], f[2 * p + 1]);
}
template <int LANES> __device__ __forceinline__ void row_barrier(uint32_t mask) {
    if (LANES == 0)
        __syncthreads();
    else
        __syncwarp(mask);
}

// How rows are shared out: threads of a CTA, CTAs of a cluster, lanes of a row in a CTA of one warp; rows that are worked on together, a
// multiple of those of a CTA; streams that are copied ahead and for how many rounds; bytes of shared memory for them.
struct Shape {
    int threads, ctas_per_row, lanes, rows_at_once;
    int streams, ahead;
    size_t ring;
    int rows_per_cta() const { return threads == 32 && ctas_per_row == 1 ? 32 / lanes : 1; }
};
// The row that a CTA's thread begins with, and its CTA's place in a cluster.
template <int LANES> __device__ __forceinline__ int first_row(const Shape &s, int &rank) {
    rank = 0;
    if constexpr (LANES > 0) return blockIdx.x * (32 / LANES) + threadIdx.x / LANES;
    if (s.ctas_per_row > 1) rank = blockIdx.x % s.ctas_per_row;
    return blockIdx.x / s.ctas_per_row;
}

// Means and 1 / deviations of two rows: the means first (0 for rms), then the squares of what is left.
template <int N, int LANES>
__device__ __forceinline__ void two_stats(const Eight (&v)[2], int kind, const Columns<N, LANES> &c, float eps, RowSum<LANES> &sum, float (&mean)[2], float (&r)[2]) {
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

// How the backward pass deals its rows out.  A unit is a run of rows of one sample (with a gate per sample, whose
// gradient is a sum over them) or of all rows.
struct Deal {
    Shape shape;
    long long samples, tokens, splits, units;
    int columns; // column sums of each cluster: weight, bias, post_weight, post_bias, scale
    int runs;    // that their partial rows are added up in first, or 1
};
// Partial rows: [rows_at_once][columns][width] of the column sums; [runs][columns][width] where those are added up in two steps; [units][width]
// of the gate's with more than one split.
struct Partials {
    float *columns, *runs, *gate;
};

constexpr int kColumns = 5;

// What is known of a call when its kernel is compiled: nothing; or that there are a branch, a norm behind it and (backward) gradients of both
// results, and that the stream's is wanted, with no gate, one per sample or one per token.  (Forward and backward, bf16, as compiled and as
// any call: 256 x 197 rows of 768, plain, 136 and 142 us, without a scale 124 and 137; 64 x 577 rows of 1024 with a gate per token 196 and
// 214, an inner norm besides 179 and 196, a gate per sample and an inner norm 150 and 190; 128 x 197 rows of 387 values, one by one, plain,
// 63 and 85, of 775 108 and 152.)
enum Form { kAny, kPlain, kGated, kToken };
inline Form form_of(const Args &a, bool backward) {
    if (!a.h || a.norm == FFCVB_NORM_NONE || (backward && (!a.dy || !a.dz || !a.dx))) return kAny;
    return a.gate_kind == FFCVB_GATE_SAMPLE ? kGated : a.gate_kind == FFCVB_GATE_TOKEN ? kToken : kPlain;
}
template <Form F> using FormOf = Int<(int)F>;
// f(packs of N, post, form): for single values the gated forms are as any call.
template <typename T, typename F> void with_form(bool wide, bool post, Form form, F &&f) {
    using Wide = Int<16 / (int)sizeof(T)>;
    auto formed = [&](auto post_norm) {
        if (!wide && form == kPlain)
            f(Int<1>{}, post_norm, FormOf<kPlain>{});
        else if (!wide)
            f(Int<1>{}, post_norm, FormOf<kAny>{});
        else if (form == kPlain)
            f(Wide{}, post_norm, FormOf<kPlain>{});
        else if (form == kGated)
            f(Wide{}, post_norm, FormOf<kGated>{});
        else if (form == kToken)
            f(Wide{}, post_norm, FormOf<kToken>{});
        else
            f(Wide{}, post_norm, FormOf<kAny>{});
    };
    if (post)
        formed(Int<1>{});
    else
        formed(Int<0>{});
}

// Shared memory that a CTA asks for at most, 213 KB (the general form backward, gated per sample, on 4096 odd columns of 32 bits), and room to the
// 227 that it may have, the static part among them.  A kernel is allowed it once and for all: the limit is the kernel's, not the call's, and
// another thread's call of it that needs less must not lower it in between.
constexpr int kMostRoom = 226 * 1024;
template <typename Kernel, typename... More>
void launch(Kernel kernel, const Shape &shape, size_t room, cudaStream_t stream, const More &...more) {
    // (what a CTA may have without being asked includes the static part)
    if (room > 40 * 1024) cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostRoom);
    cudaLaunchConfig_t how{};
    cudaLaunchAttribute with[2] = {};
    with[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    with[0].val.programmaticStreamSerializationAllowed = 1;
    with[1].id = cudaLaunchAttributeClusterDimension;
    with[1].val.clusterDim.x = shape.ctas_per_row;
    with[1].val.clusterDim.y = with[1].val.clusterDim.z = 1;
    how.gridDim = dim3(shape.rows_at_once / shape.rows_per_cta() * shape.ctas_per_row);
    how.blockDim = dim3(shape.threads);
    how.dynamicSmemBytes = room;
    how.stream = stream;
    how.attrs = with;
    how.numAttrs = shape.ctas_per_row > 1 ? 2 : 1;
    cudaLaunchKernelEx(&how, kernel, more...);
}


// wide: rows in packs of 16 bytes.
void launch_forward(const Args &a, const Shape &shape, bool wide, cudaStream_t stream);
void launch_backward(const Args &a, const Deal &deal, const Partials &part, bool wide, cudaStream_t stream);

} // namespace norms

} // namespace ffcvb
