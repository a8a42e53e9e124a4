// Group norm with an activation, of images that lie channels last, forward and backward (sm_100a).
//
// A group of a sample are its m = positions * channels / groups values.  With their mean and r = 1 / sqrt(var + eps), hat = (x - mean) r,
//   a = hat w + b,  y = act(a);  backward  da = dy act'(a),  dx = r (da w - mean(da w) - hat mean(da w hat)),  dw = sum da hat,  db = sum da.
// The means over a group are sums over its channels of w times the sums over positions of da and da hat, which the weights' gradients need too.
//
// What fits is held: some groups of a sample (channels of 64 bytes or more), at all positions, in the shared memory of a CTA or of a cluster's, so that x
// (backward x and dy) is read once.  Threads copy what they use themselves, in places of their own, and exchange moments or sums
// across the CTA and the cluster.  What does not fit is read twice, by kernels for the sums, for joining them, and for the values.
// Variances are joined from means and squares around them (of a thread's values relative to its first), which loses no digits where means are large.
#include "training.h"
#include "two.h"

#include <algorithm>
#include <type_traits>

namespace ffcvb {

// Two values of 16 bits.
template <> struct Pack<__nv_bfloat16, 2> {
    uint32_t raw;
    __device__ __forceinline__ void load(const __nv_bfloat16 *p) { raw = *reinterpret_cast<const uint32_t *>(p); }
    __device__ __forceinline__ void store(__nv_bfloat16 *p) const { *reinterpret_cast<uint32_t *>(p) = raw; }
    __device__ __forceinline__ void get(float (&v)[2]) const {
        v[0] = __uint_as_float(raw << 16);
        v[1] = __uint_as_float(raw & 0xffff0000u);
    }
    __device__ __forceinline__ void set(const float (&v)[2]) {
        const __nv_bfloat162 two = __floats2bfloat162_rn(v[0], v[1]);
        raw = *reinterpret_cast<const uint32_t *>(&two);
    }
};
template <> struct Pack<__half, 2> {
    uint32_t raw;
    __device__ __forceinline__ void load(const __half *p) { raw = *reinterpret_cast<const uint32_t *>(p); }
    __device__ __forceinline__ void store(__half *p) const { *reinterpret_cast<uint32_t *>(p) = raw; }
    __device__ __forceinline__ void get(float (&v)[2]) const {
        const float2 two = __half22float2(*reinterpret_cast<const __half2 *>(&raw));
        v[0] = two.x, v[1] = two.y;
    }
    __device__ __forceinline__ void set(const float (&v)[2]) {
        const __half2 two = __floats2half2_rn(v[0], v[1]);
        raw = *reinterpret_cast<const uint32_t *>(&two);
    }
};

namespace {

constexpr int kThreads = 256;
constexpr int kMostGroups = 32; // of a CTA
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float exp_of(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * kLog2e));
    return y;
}

template <int N> __device__ __forceinline__ void activate(float (&v)[N], int kind) {
    if (kind == FFCVB_ACT_SILU) {
#pragma unroll
        for (int j = 0; j < N; j++) v[j] = __fdividef(v[j], 1.0f + exp_of(-v[j]));
    } else if (kind == FFCVB_ACT_GELU) {
#pragma unroll
        for (int j = 0; j < N; j++) v[j] = 0.5f * v[j] * (1.0f + erff(v[j] * 0.70710678118654752f));
    } else if (kind == FFCVB_ACT_RELU) {
#pragma unroll
        for (int j = 0; j < N; j++) v[j] = v[j] > 0.0f || v[j] != v[j] ? v[j] : 0.0f;
    }
}
// act'(a) dy in the place of dy
template <int N> __device__ __forceinline__ void slope(float (&d)[N], const float (&a)[N], int kind) {
    if (kind == FFCVB_ACT_SILU) {
#pragma unroll
        for (int j = 0; j < N; j++) {
            const float gate = __fdividef(1.0f, 1.0f + exp_of(-a[j]));
            d[j] *= gate * fmaf(a[j], 1.0f - gate, 1.0f);
        }
    } else if (kind == FFCVB_ACT_GELU) {
#pragma unroll
        for (int j = 0; j < N; j++) d[j] *= fmaf(0.39894228040143268f * a[j], exp_of(-0.5f * a[j] * a[j]), 0.5f * (1.0f + erff(a[j] * 0.70710678118654752f)));
    } else if (kind == FFCVB_ACT_RELU) {
#pragma unroll
        for (int j = 0; j < N; j++) d[j] = a[j] > 0.0f ? d[j] : 0.0f;
    }
}

// How many, their mean, and the sum of squares around it.
struct Moments {
    float n, mean, squares;
    __device__ __forceinline__ void join(Moments o) {
        const float all = n + o.n, share = o.n == 0.0f ? 0.0f : o.n / all, apart = o.mean - mean;
        squares += o.squares + apart * apart * n * share;
        mean += apart * share;
        n = all;
    }
    // of a warp; lane 0 has the result
    __device__ __forceinline__ void join_lanes() {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
            join(Moments{__shfl_down_sync(0xffffffffu, n, o), __shfl_down_sync(0xffffffffu, mean, o), __shfl_down_sync(0xffffffffu, squares, o)});
    }
    __device__ __forceinline__ float rate(float eps) const { return rsqrtf(squares / n + eps); }
};

// Values of a thread, relative to its first one.
template <int W> struct Collected {
    float first, sum, squares;
    int rows;
    __device__ __forceinline__ void add(const float (&v)[W]) {
        if (rows++ == 0) first = v[0], sum = squares = 0.0f;
#pragma unroll
        for (int j = 0; j < W; j++) {
            const float d = v[j] - first;
            sum += d;
            squares = fmaf(d, d, squares);
        }
    }
    __device__ __forceinline__ Moments moments() const {
        if (rows == 0) return Moments{0.0f, 0.0f, 0.0f};
        const float n = (float)(rows * W), mean = sum / n;
        const float around = squares - sum * mean;
        return Moments{n, first + mean, around < 0.0f ? 0.0f : around}; // (NaN stays)
    }
};

// W neighbouring parameters, or what stands for them.
template <int W> __device__ __forceinline__ void parameters(float (&v)[W], const void *from, int type, long long c, float other) {
#pragma unroll
    for (int j = 0; j < W; j++)
        v[j] = !from                        ? other
               : type == FFCVB_TYPE_F32     ? static_cast<const float *>(from)[c + j]
               : type == FFCVB_TYPE_F16     ? to_float(static_cast<const __half *>(from)[c + j])
                                            : to_float(static_cast<const __nv_bfloat16 *>(from)[c + j]);
}

// A pack that a thread has copied for itself.
template <typename T, int W> __device__ __forceinline__ void copy_pack(Pack<T, W> *to, const T *from) {
    constexpr int BYTES = W * sizeof(T);
    const uint32_t at = (uint32_t)__cvta_generic_to_shared(to);
    if constexpr (BYTES == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(from) : "memory");
    else if constexpr (BYTES >= 4)
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(at), "l"(from), "n"(BYTES) : "memory");
    else
        to->load(from);
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_begun() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() { asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void store_there(const void *mine, uint32_t rank, float v) {
    uint32_t at;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(mine)), "r"(rank));
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at), "f"(v) : "memory");
}

// ---- held: a CTA or a cluster has some groups of a sample at all positions ---------------------------------------------

// Groups of a CTA, packs of a position in them, of which `lanes` positions at once; positions of a CTA; CTAs of a cluster.
struct Deal {
    int groups, packs, lanes, rows, ctas;
};

template <typename T, int W>
__global__ void __launch_bounds__(kThreads) held_forward_kernel(const __grid_constant__ ffcvb_group_norm_args a, const Deal deal) {
    __shared__ float s_moments[3][kThreads];
    __shared__ Moments s_there[8][kMostGroups]; // of the cluster's CTAs
    extern __shared__ uint4 s_held[];
    wait_for_previous();
    let_next_begin();
    const uint32_t rank = deal.ctas > 1 ? cluster_rank() : 0;
    if (deal.ctas > 1) cluster_begun();
    const int per = (int)(a.channels / a.groups), blocks = (int)a.groups / deal.groups, unit = blockIdx.x / deal.ctas;
    const long long sample = unit / blocks;
    const int group0 = unit % blocks * deal.groups, row = threadIdx.x / deal.packs, pack = threadIdx.x % deal.packs;
    const int first = (int)rank * deal.rows, last = min(first + deal.rows, (int)a.positions);
    const int group = pack * W / per, channel = group0 * per + pack * W;
    const bool used = row < deal.lanes;
    const T *x = static_cast<const T *>(a.x) + sample * a.x_sample + channel;
    Pack<T, W> *held = reinterpret_cast<Pack<T, W> *>(s_held) + threadIdx.x;
    if (used) {
        Pack<T, W> *to = held;
        for (int r = first + row; r < last; r += deal.lanes, to += kThreads) copy_pack(to, x + r * a.x_position);
    }
    float w[W], b[W];
    if (used) {
        parameters(w, a.weight, a.param_type, channel, 1.0f);
        parameters(b, a.bias, a.param_type, channel, 0.0f);
    }
    copies_done();
    Collected<W> values{0.0f, 0.0f, 0.0f, 0};
    if (used) {
        const Pack<T, W> *from = held;
        for (int r = first + row; r < last; r += deal.lanes, from += kThreads) {
            float v[W];
            from->get(v);
            values.add(v);
        }
    }
    const Moments mine = values.moments();
    s_moments[0][threadIdx.x] = mine.n, s_moments[1][threadIdx.x] = mine.mean, s_moments[2][threadIdx.x] = mine.squares;
    __syncthreads();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, each = per / W; // packs of a group
    if (deal.ctas > 1) cluster_wait(); // all have begun
    for (int g = warp; g < deal.groups; g += kThreads / 32) {
        Moments all{0.0f, 0.0f, 0.0f};
        for (int e = lane; e < deal.lanes * each; e += 32) {
            const int t = e / each * deal.packs + g * each + e % each;
            all.join(Moments{s_moments[0][t], s_moments[1][t], s_moments[2][t]});
        }
        all.join_lanes();
        const float n = __shfl_sync(0xffffffffu, all.n, 0), mean = __shfl_sync(0xffffffffu, all.mean, 0), squares = __shfl_sync(0xffffffffu, all.squares, 0);
        if (lane < deal.ctas) {
            Moments *to = &s_there[rank][g];
            if (deal.ctas == 1) {
                *to = Moments{n, mean, squares};
            } else {
                store_there(&to->n, lane, n);
                store_there(&to->mean, lane, mean);
                store_there(&to->squares, lane, squares);
            }
        }
    }
    if (deal.ctas > 1)
        cluster_sync();
    else
        __syncthreads();
    if (!used) return;
    Moments all = s_there[0][group];
    for (int k = 1; k < deal.ctas; k++) all.join(s_there[k][group]);
    const float rate = all.rate(a.eps);
    if (rank == 0 && row == 0 && pack % each == 0) reinterpret_cast<float2 *>(a.stats)[sample * a.groups + group0 + group] = make_float2(all.mean, rate);
#pragma unroll
    for (int j = 0; j < W; j++) w[j] *= rate;
    T *y = static_cast<T *>(a.y) + sample * a.positions * a.channels + channel;
    const Pack<T, W> *from = held;
    for (int r = first + row; r < last; r += deal.lanes, from += kThreads) {
        float v[W];
        from->get(v);
#pragma unroll
        for (int j = 0; j < W; j++) v[j] = fmaf(v[j] - all.mean, w[j], b[j]);
        activate(v, a.activation);
        Pack<T, W> out;
        out.set(v);
        out.store(y + r * a.channels);
    }
}

// Sums over positions of da and da hat: of a thread's channels joined over the rows of the CTA, in s_sums[channel]; `s_all` is room for all threads'.
template <int W> __device__ __forceinline__ void channel_sums(const float2 (&mine)[W], bool used, int row, int pack, int lanes, int packs, float2 *s_all, float2 *s_sums) {
    const int channels = packs * W;
    if (used)
#pragma unroll
        for (int j = 0; j < W; j++) s_all[row * channels + pack * W + j] = mine[j];
    __syncthreads();
    // lanes are halved until one is left, always in the same order
    for (int n = lanes; n > 1;) {
        const int half = (n + 1) / 2;
        for (int i = threadIdx.x; i < (n - half) * channels; i += kThreads) {
            s_all[i].x += s_all[i + half * channels].x;
            s_all[i].y += s_all[i + half * channels].y;
        }
        n = half;
        __syncthreads();
    }
    for (int i = threadIdx.x; i < channels; i += kThreads) s_sums[i] = s_all[i];
}

// room: 2 * kThreads * W floats for sums, of the cluster's CTAs as many channels' as there are; then x and dy
template <typename T, int W>
__global__ void __launch_bounds__(kThreads) held_backward_kernel(const __grid_constant__ ffcvb_group_norm_args a, const Deal deal, float2 *sums) {
    __shared__ float2 s_group[kMostGroups];
    extern __shared__ uint4 s_held[];
    wait_for_previous();
    let_next_begin();
    const uint32_t rank = deal.ctas > 1 ? cluster_rank() : 0;
    if (deal.ctas > 1) cluster_begun();
    const int per = (int)(a.channels / a.groups), blocks = (int)a.groups / deal.groups, unit = blockIdx.x / deal.ctas;
    const long long sample = unit / blocks;
    const int group0 = unit % blocks * deal.groups, row = threadIdx.x / deal.packs, pack = threadIdx.x % deal.packs, channels = deal.packs * W;
    const int first = (int)rank * deal.rows, last = min(first + deal.rows, (int)a.positions);
    const int group = pack * W / per, channel = group0 * per + pack * W;
    const bool used = row < deal.lanes;
    const T *x = static_cast<const T *>(a.x) + sample * a.x_sample + channel, *dy = static_cast<const T *>(a.dy) + sample * a.dy_sample + channel;
    float2 *s_all = reinterpret_cast<float2 *>(s_held), *s_there = s_all + deal.lanes * channels; // [ctas][channels]
    Pack<T, W> *held = reinterpret_cast<Pack<T, W> *>(s_held + ((deal.lanes + deal.ctas) * channels + 1) / 2) + threadIdx.x;
    if (used) {
        Pack<T, W> *to = held;
        for (int r = first + row; r < last; r += deal.lanes, to += 2 * kThreads) {
            copy_pack(to, x + r * a.x_position);
            copy_pack(to + kThreads, dy + r * a.dy_position);
        }
    }
    float w[W], b[W], mean = 0.0f, rate = 0.0f;
    float2 mine[W];
#pragma unroll
    for (int j = 0; j < W; j++) mine[j] = make_float2(0.0f, 0.0f);
    if (used) {
        parameters(w, a.weight, a.param_type, channel, 1.0f);
        parameters(b, a.bias, a.param_type, channel, 0.0f);
        const float2 stats = reinterpret_cast<const float2 *>(a.stats)[sample * a.groups + group0 + group];
        mean = stats.x, rate = stats.y;
    }
    copies_done();
    // hat and da of a row
    auto row_of = [&](const Pack<T, W> *from, float(&hat)[W], float(&da)[W]) {
        from->get(hat);
        from[kThreads].get(da);
        float v[W];
#pragma unroll
        for (int j = 0; j < W; j++) {
            hat[j] = (hat[j] - mean) * rate;
            v[j] = fmaf(hat[j], w[j], b[j]);
        }
        slope(da, v, a.activation);
    };
    if (used) {
        const Pack<T, W> *from = held;
        for (int r = first + row; r < last; r += deal.lanes, from += 2 * kThreads) {
            float hat[W], da[W];
            row_of(from, hat, da);
#pragma unroll
            for (int j = 0; j < W; j++) {
                mine[j].x += da[j];
                mine[j].y = fmaf(da[j], hat[j], mine[j].y);
            }
        }
    }
    channel_sums<W>(mine, used, row, pack, deal.lanes, deal.packs, s_all, s_there + (deal.ctas > 1 ? (int)rank * channels : 0));
    if (deal.ctas > 1) {
        __syncthreads();
        cluster_wait(); // all have begun
        for (int i = threadIdx.x; i < channels * deal.ctas; i += kThreads) {
            const int c = i % channels, to = i / channels;
            float2 *at = s_there + rank * channels + c;
            if (to == (int)rank) continue;
            const float2 v = *at;
            store_there(&at->x, to, v.x);
            store_there(&at->y, to, v.y);
        }
        cluster_sync();
        for (int i = threadIdx.x; i < channels; i += kThreads) {
            float2 all = s_there[i];
            for (int k = 1; k < deal.ctas; k++) {
                all.x += s_there[k * channels + i].x;
                all.y += s_there[k * channels + i].y;
            }
            s_all[i] = all;
        }
    } else {
        for (int i = threadIdx.x; i < channels; i += kThreads) s_all[i] = s_there[i]; // (each its own)
    }
    __syncthreads();
    if (rank == 0)
        for (int i = threadIdx.x; i < channels; i += kThreads) sums[sample * a.channels + group0 * per + i] = s_all[i];
    for (int g = threadIdx.x >> 5; g < deal.groups; g += kThreads / 32) {
        float2 all = make_float2(0.0f, 0.0f);
        for (int c = threadIdx.x & 31; c < per; c += 32) {
            float one[1];
            parameters(one, a.weight, a.param_type, group0 * per + g * per + c, 1.0f);
            all.x = fmaf(one[0], s_all[g * per + c].x, all.x);
            all.y = fmaf(one[0], s_all[g * per + c].y, all.y);
        }
        const float over = 1.0f / ((float)a.positions * (float)per);
        all.x = warp_sum(all.x) * over;
        all.y = warp_sum(all.y) * over;
        if ((threadIdx.x & 31) == 0) s_group[g] = all;
    }
    __syncthreads();
    if (!used || !a.dx) return;
    const float2 less = s_group[group];
    T *dx = static_cast<T *>(a.dx) + sample * a.positions * a.channels + channel;
    const Pack<T, W> *from = held;
    for (int r = first + row; r < last; r += deal.lanes, from += 2 * kThreads) {
        float hat[W], da[W];
        row_of(from, hat, da);
#pragma unroll
        for (int j = 0; j < W; j++) da[j] = rate * (fmaf(da[j], w[j], -less.x) - hat[j] * less.y);
        Pack<T, W> out;
        out.set(da);
        out.store(dx + r * a.channels);
    }
}

// ---- not held: sums of slabs of positions, joined; then the values -------------------------------------------------------

// Packs of a position, of which a CTA has `columns`, and `lanes` positions at once; positions of a slab, and slabs.  Samples from `sample` on.
struct Slabs {
    int packs, columns, lanes, rows, slabs;
    int64_t sample;
};

struct Place {
    int row, pack, slab, first, last;
    long long sample;
    bool used;
};
// `backwards`: the slabs that were read last are still in the caches and come first.
__device__ __forceinline__ Place place_of(const Slabs &s, int positions, bool backwards) {
    Place p;
    p.row = threadIdx.x / s.columns;
    p.pack = blockIdx.y * s.columns + threadIdx.x % s.columns;
    const long long n = backwards ? (long long)gridDim.x - 1 - blockIdx.x : blockIdx.x;
    p.slab = (int)(n % s.slabs);
    p.sample = s.sample + n / s.slabs;
    p.first = p.slab * s.rows;
    p.last = min(p.first + s.rows, positions);
    p.used = p.row < s.lanes && p.pack < s.packs;
    return p;
}

template <typename T, int W>
__global__ void __launch_bounds__(kThreads) moments_kernel(const __grid_constant__ ffcvb_group_norm_args a, const Slabs s, float2 *parts) {
    __shared__ Moments s_moments[kThreads];
    wait_for_previous();
    let_next_begin();
    const Place p = place_of(s, (int)a.positions, false);
    Collected<W> values{0.0f, 0.0f, 0.0f, 0};
    if (p.used) {
        const T *x = static_cast<const T *>(a.x) + p.sample * a.x_sample + p.pack * W;
#pragma unroll 4
        for (int r = p.first + p.row; r < p.last; r += s.lanes) {
            Pack<T, W> pack;
            float v[W];
            pack.load(x + r * a.x_position);
            pack.get(v);
            values.add(v);
        }
    }
    s_moments[threadIdx.x] = values.moments();
    __syncthreads();
    if (p.row != 0 || !p.used) return;
    Moments all = s_moments[threadIdx.x];
    for (int k = 1; k < s.lanes; k++) all.join(s_moments[k * s.columns + threadIdx.x]);
    parts[(p.sample * s.slabs + p.slab) * s.packs + p.pack] = make_float2(all.mean, all.squares);
}

// One warp per group.
template <int W> __global__ void __launch_bounds__(kThreads) join_moments_kernel(const __grid_constant__ ffcvb_group_norm_args a, const Slabs s, int samples, const float2 *parts) {
    wait_for_previous();
    let_next_begin();
    const long long n = blockIdx.x * (kThreads / 32ll) + (threadIdx.x >> 5);
    if (n >= samples * a.groups) return;
    const long long sample = s.sample + n / a.groups;
    const int group = (int)(n % a.groups), each = (int)(a.channels / a.groups) / W;
    Moments all{0.0f, 0.0f, 0.0f};
    for (long long e = threadIdx.x & 31; e < (long long)s.slabs * each; e += 32) {
        const int slab = (int)(e / each);
        const float2 part = parts[(sample * s.slabs + slab) * s.packs + group * each + e % each];
        all.join(Moments{(float)(min(s.rows, (int)a.positions - slab * s.rows) * W), part.x, part.y});
    }
    all.join_lanes();
    if ((threadIdx.x & 31) == 0) reinterpret_cast<float2 *>(a.stats)[sample * a.groups + group] = make_float2(all.mean, all.rate(a.eps));
}

template <typename T, int W>
__global__ void __launch_bounds__(kThreads) values_kernel(const __grid_constant__ ffcvb_group_norm_args a, const Slabs s) {
    wait_for_previous();
    let_next_begin();
    const Place p = place_of(s, (int)a.positions, true);
    if (!p.used) return;
    const int channel = p.pack * W, group = channel / (int)(a.channels / a.groups);
    float w[W], b[W];
    parameters(w, a.weight, a.param_type, channel, 1.0f);
    parameters(b, a.bias, a.param_type, channel, 0.0f);
    const float2 stats = reinterpret_cast<const float2 *>(a.stats)[p.sample * a.groups + group];
#pragma unroll
    for (int j = 0; j < W; j++) w[j] *= stats.y;
    const T *x = static_cast<const T *>(a.x) + p.sample * a.x_sample + channel;
    T *y = static_cast<T *>(a.y) + p.sample * a.positions * a.channels + channel;
#pragma unroll 4
    for (int r = p.first + p.row; r < p.last; r += s.lanes) {
        Pack<T, W> pack;
        float v[W];
        pack.load(x + r * a.x_position);
        pack.get(v);
#pragma unroll
        for (int j = 0; j < W; j++) v[j] = fmaf(v[j] - stats.x, w[j], b[j]);
        activate(v, a.activation);
        pack.set(v);
        pack.store(y + r * a.channels);
    }
}

// hat and da of W channels.
template <typename T, int W> struct Back {
    float w[W], b[W], mean, rate;
    int kind;
    __device__ __forceinline__ Back(const ffcvb_group_norm_args &a, long long sample, int channel) : kind(a.activation) {
        parameters(w, a.weight, a.param_type, channel, 1.0f);
        parameters(b, a.bias, a.param_type, channel, 0.0f);
        const float2 stats = reinterpret_cast<const float2 *>(a.stats)[sample * a.groups + channel / (int)(a.channels / a.groups)];
        mean = stats.x, rate = stats.y;
    }
    __device__ __forceinline__ void row(const T *x, const T *dy, float (&hat)[W], float (&da)[W]) const {
        Pack<T, W> one, other;
        one.load(x);
        other.load(dy);
        one.get(hat);
        other.get(da);
        float v[W];
#pragma unroll
        for (int j = 0; j < W; j++) {
            hat[j] = (hat[j] - mean) * rate;
            v[j] = fmaf(hat[j], w[j], b[j]);
        }
        slope(da, v, kind);
    }
};

// parts: [samples][slabs][channels]
template <typename T, int W>
__global__ void __launch_bounds__(kThreads) sums_kernel(const __grid_constant__ ffcvb_group_norm_args a, const Slabs s, float2 *parts) {
    __shared__ float2 s_all[kThreads * W];
    wait_for_previous();
    let_next_begin();
    const Place p = place_of(s, (int)a.positions, false);
    float2 mine[W];
#pragma unroll
    for (int j = 0; j < W; j++) mine[j] = make_float2(0.0f, 0.0f);
    if (p.used) {
        const int channel = p.pack * W;
        const Back<T, W> back(a, p.sample, channel);
        const T *x = static_cast<const T *>(a.x) + p.sample * a.x_sample + channel, *dy = static_cast<const T *>(a.dy) + p.sample * a.dy_sample + channel;
#pragma unroll 2
        for (int r = p.first + p.row; r < p.last; r += s.lanes) {
            float hat[W], da[W];
            back.row(x + r * a.x_position, dy + r * a.dy_position, hat, da);
#pragma unroll
            for (int j = 0; j < W; j++) {
                mine[j].x += da[j];
                mine[j].y = fmaf(da[j], hat[j], mine[j].y);
            }
        }
    }
    float2 *to = parts + (p.sample * s.slabs + p.slab) * a.channels + blockIdx.y * s.columns * W;
    const int channels = s.columns * W, there = min(channels, (int)a.channels - (int)blockIdx.y * channels);
    if (p.row < s.lanes)
#pragma unroll
        for (int j = 0; j < W; j++) s_all[p.row * channels + threadIdx.x % s.columns * W + j] = mine[j];
    __syncthreads();
    for (int c = threadIdx.x; c < there; c += kThreads) {
        float2 all = s_all[c];
        for (int k = 1; k < s.lanes; k++) {
            all.x += s_all[k * channels + c].x;
            all.y += s_all[k * channels + c].y;
        }
        to[c] = all;
    }
}

// A CTA per group: its channels' sums, [samples][channels], and its means, [samples][groups].
__global__ void __launch_bounds__(kThreads) join_sums_kernel(const __grid_constant__ ffcvb_group_norm_args a, const Slabs s, const float2 *parts, float2 *sums, float2 *means) {
    __shared__ float2 s_part[kThreads / 32];
    wait_for_previous();
    let_next_begin();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, per = (int)(a.channels / a.groups), group = (int)(blockIdx.x % a.groups);
    const long long sample = s.sample + blockIdx.x / a.groups;
    float2 mean = make_float2(0.0f, 0.0f);
    for (int c = group * per + warp; c < (group + 1) * per; c += kThreads / 32) {
        float2 all = make_float2(0.0f, 0.0f);
        for (int k = lane; k < s.slabs; k += 32) {
            const float2 part = parts[(sample * s.slabs + k) * a.channels + c];
            all.x += part.x;
            all.y += part.y;
        }
        all.x = warp_sum(all.x);
        all.y = warp_sum(all.y);
        float w[1];
        parameters(w, a.weight, a.param_type, c, 1.0f);
        mean.x = fmaf(w[0], all.x, mean.x);
        mean.y = fmaf(w[0], all.y, mean.y);
        if (lane == 0) sums[sample * a.channels + c] = all;
    }
    if (lane == 0) s_part[warp] = mean;
    __syncthreads();
    if (threadIdx.x) return;
    for (int k = 1; k < kThreads / 32; k++) {
        mean.x += s_part[k].x;
        mean.y += s_part[k].y;
    }
    const float over = 1.0f / ((float)a.positions * (float)per);
    means[sample * a.groups + group] = make_float2(mean.x * over, mean.y * over);
}

template <typename T, int W>
__global__ void __launch_bounds__(kThreads) gradient_kernel(const __grid_constant__ ffcvb_group_norm_args a, const Slabs s, const float2 *means) {
    wait_for_previous();
    let_next_begin();
    const Place p = place_of(s, (int)a.positions, true);
    if (!p.used) return;
    const int channel = p.pack * W;
    const Back<T, W> back(a, p.sample, channel);
    const float2 less = means[p.sample * a.groups + channel / (int)(a.channels / a.groups)];
    const T *x = static_cast<const T *>(a.x) + p.sample * a.x_sample + channel, *dy = static_cast<const T *>(a.dy) + p.sample * a.dy_sample + channel;
    T *dx = static_cast<T *>(a.dx) + p.sample * a.positions * a.channels + channel;
#pragma unroll 2
    for (int r = p.first + p.row; r < p.last; r += s.lanes) {
        float hat[W], da[W];
        back.row(x + r * a.x_position, dy + r * a.dy_position, hat, da);
#pragma unroll
        for (int j = 0; j < W; j++) da[j] = back.rate * (fmaf(da[j], back.w[j], -less.x) - hat[j] * less.y);
        Pack<T, W> out;
        out.set(da);
        out.store(dx + r * a.channels);
    }
}

// The parameters' gradients: samples' sums added up, 32 channels per CTA.
__global__ void __launch_bounds__(kThreads) samples_kernel(const __grid_constant__ ffcvb_group_norm_args a, const float2 *sums) {
    __shared__ float2 s_part[kThreads / 32][32];
    wait_for_previous();
    let_next_begin();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long c = blockIdx.x * 32ll + lane;
    float2 all = make_float2(0.0f, 0.0f);
    if (c < a.channels)
#pragma unroll 4
        for (long long n = warp; n < a.samples; n += kThreads / 32) {
            const float2 part = sums[n * a.channels + c];
            all.x += part.x;
            all.y += part.y;
        }
    s_part[warp][lane] = all;
    __syncthreads();
    if (warp || c >= a.channels) return;
    for (int k = 1; k < kThreads / 32; k++) {
        all.x += s_part[k][lane].x;
        all.y += s_part[k][lane].y;
    }
    auto put = [&](void *to, float v) {
        if (!to) return;
        if (a.param_type == FFCVB_TYPE_F32)
            static_cast<float *>(to)[c] = v;
        else if (a.param_type == FFCVB_TYPE_F16)
            static_cast<__half *>(to)[c] = from_float<__half>(v);
        else
            static_cast<__nv_bfloat16 *>(to)[c] = from_float<__nv_bfloat16>(v);
    };
    put(a.dbias, all.x);
    put(a.dweight, all.y);
}

// ---- the host's part -------------------------------------------------------------------------------------------------

// Bytes that a CTA holds at most: two of them on an SM; and what it holds rather, so that four are.
constexpr int64_t kMostHeld = 100 * 1024, kHeld = 52 * 1024;
// Bytes of neighbouring channels that a CTA reads at least, where there are as many.
constexpr int64_t kNeighbours = 64;
// Bytes of x of a pass over all its slabs, before they are read again: what the caches keep.
constexpr int64_t kCached = 40ll << 20;

// Values of a pack: all of one group, and where they begin as their size has it.
int width_of(const ffcvb_group_norm_args &a, bool backward) {
    const int size = type_size(a.type);
    int w = 16 / size;
    auto fits = [&](const void *p, int64_t sample, int64_t position) {
        return reinterpret_cast<uintptr_t>(p) % (w * size) == 0 && (a.samples <= 1 || sample % w == 0) && (a.positions <= 1 || position % w == 0);
    };
    for (; w > 1; w /= 2)
        if (a.channels / a.groups % w == 0 && fits(a.x, a.x_sample, a.x_position) &&
            (backward ? fits(a.dy, a.dy_sample, a.dy_position) && (!a.dx || fits(a.dx, 0, 0)) : fits(a.y, 0, 0)))
            break;
    return w;
}

struct Plan {
    int width;
    bool held;
    Deal deal;
    int64_t room;     // bytes of shared memory
    Slabs slabs;
    int64_t samples;  // at once
    int64_t parts, means, sums, bytes; // offsets in the workspace
};

Plan plan_of(const ffcvb_group_norm_args &a, bool backward) {
    Plan p{};
    const int size = type_size(a.type), w = p.width = width_of(a, backward);
    const int64_t per = a.channels / a.groups;
    Deal &d = p.deal;
    d.groups = 1;
    while (d.groups * 2 <= kMostGroups && a.groups % (d.groups * 2) == 0 && d.groups * per * size < kNeighbours) d.groups *= 2;
    const int64_t packs = d.groups * per / w;
    if (packs <= kThreads) {
        d.packs = (int)packs;
        d.lanes = (int)std::min<int64_t>(kThreads / packs, std::max<int64_t>(a.positions, 1));
        auto room_of = [&](int ctas) {
            const int64_t rows = (a.positions + ctas - 1) / ctas, turns = (rows + d.lanes - 1) / d.lanes;
            return turns * kThreads * w * size * (backward ? 2 : 1) + (backward ? ((d.lanes + ctas) * packs * w + 1) / 2 * 16 : 0);
        };
        for (d.ctas = 1; d.ctas < 8 && room_of(d.ctas) > kHeld; d.ctas *= 2) {}
        p.room = room_of(d.ctas);
        p.held = p.room <= kMostHeld;
        d.rows = (int)((a.positions + d.ctas - 1) / d.ctas);
        p.held &= a.samples * (a.groups / d.groups) * d.ctas <= INT32_MAX;
    }
    Slabs &s = p.slabs;
    s.packs = (int)(a.channels / w);
    s.columns = std::min(s.packs, kThreads);
    s.lanes = std::max(1, kThreads / s.columns);
    // slabs of 16 to 64 positions of a thread, as many as bring two rounds of CTAs to all SMs
    const int64_t all = a.samples * ((s.packs + s.columns - 1) / s.columns);
    int64_t turns = a.positions * all / std::max<int64_t>(1, (int64_t)s.lanes * kSms * 16);
    turns = std::clamp<int64_t>(turns, 8, 64);
    s.rows = (int)std::min<int64_t>(a.positions, turns * s.lanes);
    s.slabs = s.rows ? (int)((a.positions + s.rows - 1) / s.rows) : 0;
    const int64_t sample_bytes = a.positions * a.channels * size * (backward ? 2 : 1);
    p.samples = std::clamp<int64_t>(kCached / std::max<int64_t>(1, sample_bytes), 1, a.samples);
    int64_t at = 0;
    auto take = [&](bool wanted, int64_t bytes) {
        const int64_t here = at;
        if (wanted) at += (bytes + 255) / 256 * 256;
        return here;
    };
    p.parts = take(!p.held, a.samples * s.slabs * (backward ? a.channels : s.packs) * 8);
    p.means = take(!p.held && backward, a.samples * a.groups * 8);
    p.sums = take(backward, a.samples * a.channels * 8);
    p.bytes = at;
    return p;
}

const char *wrong(const ffcvb_group_norm_args &a, bool backward) {
    auto known = [](int type) { return type == FFCVB_TYPE_F32 || type == FFCVB_TYPE_F16 || type == FFCVB_TYPE_BF16; };
    if (!known(a.type) || !known(a.param_type)) return "bad type";
    if (a.samples < 0 || a.positions < 0 || a.channels < 1 || a.groups < 1 || a.groups > a.channels || a.channels % a.groups != 0) return "bad size";
    if (a.samples > 1 << 24 || a.positions > 1 << 30 || a.channels > 1 << 20 || a.samples * a.groups > INT32_MAX) return "bad size";
    if (a.x_sample < 0 || a.x_position < 0 || a.dy_sample < 0 || a.dy_position < 0) return "bad stride";
    if (a.activation < FFCVB_ACT_NONE || a.activation > FFCVB_ACT_GELU || !(a.eps >= 0.0f)) return "bad argument";
    if (a.samples > 0 && a.positions > 0 && (!a.x || !a.stats || (backward ? !a.dy : !a.y))) return "an address is missing";
    if (backward && !a.dx && !a.dweight && !a.dbias) return "nothing to do";
    return nullptr;
}

// Calls f with a value of the type, and the width, of a call's packs.
template <typename T, typename F> void with_width(int w, F &&f) {
    if constexpr (sizeof(T) == 2)
        if (w == 8) return f(T{}, std::integral_constant<int, 8>{});
    if (w == 4) return f(T{}, std::integral_constant<int, 4>{});
    if (w == 2) return f(T{}, std::integral_constant<int, 2>{});
    f(T{}, std::integral_constant<int, 1>{});
}

template <typename... Params, typename... Given> void launch_cluster(void (*kernel)(Params...), int64_t ctas, int cluster, int64_t room, cudaStream_t stream, Given &&...given) {
    cudaLaunchConfig_t how{};
    cudaLaunchAttribute with[2] = {};
    with[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    with[0].val.programmaticStreamSerializationAllowed = 1;
    with[1].id = cudaLaunchAttributeClusterDimension;
    with[1].val.clusterDim.x = cluster;
    with[1].val.clusterDim.y = with[1].val.clusterDim.z = 1;
    how.gridDim = dim3((unsigned)ctas);
    how.blockDim = dim3(kThreads);
    how.dynamicSmemBytes = room;
    how.stream = stream;
    how.attrs = with;
    how.numAttrs = cluster > 1 ? 2 : 1;
    if (room > 16 * 1024) {
        // (the limit is the kernel's, not the call's: another thread's call that needs less must not lower it)
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMostHeld);
        cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    }
    cudaLaunchKernelEx(&how, kernel, static_cast<Params>(given)...);
}

void run_forward(const ffcvb_group_norm_args &a, uint8_t *room, cudaStream_t st) {
    const Plan p = plan_of(a, false);
    with_type(a.type, [&](auto zero) {
        with_width<decltype(zero)>(p.width, [&](auto of, auto width) {
            using T = decltype(of);
            constexpr int W = decltype(width)::value;
            if (p.held) {
                launch_cluster(held_forward_kernel<T, W>, a.samples * (a.groups / p.deal.groups) * p.deal.ctas, p.deal.ctas, p.room, st, a, p.deal);
                return;
            }
            float2 *parts = reinterpret_cast<float2 *>(room + p.parts);
            Slabs s = p.slabs;
            for (s.sample = 0; s.sample < a.samples; s.sample += p.samples) {
                const int64_t samples = std::min(p.samples, a.samples - s.sample);
                const dim3 grid((unsigned)(samples * s.slabs), (unsigned)((s.packs + s.columns - 1) / s.columns));
                launch_early(moments_kernel<T, W>, grid, kThreads, 0, st, a, s, parts);
                launch_early(join_moments_kernel<W>, (unsigned)((samples * a.groups + 7) / 8), kThreads, 0, st, a, s, (int)samples, parts);
                launch_early(values_kernel<T, W>, grid, kThreads, 0, st, a, s);
            }
        });
    });
}

void run_backward(const ffcvb_group_norm_args &a, uint8_t *room, cudaStream_t st) {
    const Plan p = plan_of(a, true);
    float2 *sums = reinterpret_cast<float2 *>(room + p.sums);
    with_type(a.type, [&](auto zero) {
        with_width<decltype(zero)>(p.width, [&](auto of, auto width) {
            using T = decltype(of);
            constexpr int W = decltype(width)::value;
            if (p.held) {
                launch_cluster(held_backward_kernel<T, W>, a.samples * (a.groups / p.deal.groups) * p.deal.ctas, p.deal.ctas, p.room, st, a, p.deal, sums);
                return;
            }
            float2 *parts = reinterpret_cast<float2 *>(room + p.parts), *means = reinterpret_cast<float2 *>(room + p.means);
            Slabs s = p.slabs;
            for (s.sample = 0; s.sample < a.samples; s.sample += p.samples) {
                const int64_t samples = std::min(p.samples, a.samples - s.sample);
                const dim3 grid((unsigned)(samples * s.slabs), (unsigned)((s.packs + s.columns - 1) / s.columns));
                launch_early(sums_kernel<T, W>, grid, kThreads, 0, st, a, s, parts);
                launch_early(join_sums_kernel, (unsigned)(samples * a.groups), kThreads, 0, st, a, s, parts, sums, means);
                if (a.dx) launch_early(gradient_kernel<T, W>, grid, kThreads, 0, st, a, s, means);
            }
        });
    });
    if (a.dweight || a.dbias) launch_early(samples_kernel, (unsigned)((a.channels + 31) / 32), kThreads, 0, st, a, sums);
}

int call(const ffcvb_group_norm_args *args, void *workspace, void *stream, bool backward) {
    const char *name = backward ? "ffcvb_group_norm_backward" : "ffcvb_group_norm";
    if (!args) return training_fail(FFCVB_E_ARG, "%s: no arguments", name);
    const ffcvb_group_norm_args &a = *args;
    if (const char *what = wrong(a, backward)) return training_fail(FFCVB_E_ARG, "%s: %s", name, what);
    const bool some = a.samples > 0 && a.positions > 0;
    if (some && plan_of(a, backward).bytes > 0 && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15))) return training_fail(FFCVB_E_ARG, "%s: no workspace", name);
    OnDevice here(a.device);
    if (!here.ok()) return training_fail(FFCVB_E_NODEVICE, "%s: no device %d", name, a.device);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (some) {
        (backward ? run_backward : run_forward)(a, static_cast<uint8_t *>(workspace), st);
    } else if (backward) {
        if (a.dweight) cudaMemsetAsync(a.dweight, 0, (size_t)(a.channels * type_size(a.param_type)), st);
        if (a.dbias) cudaMemsetAsync(a.dbias, 0, (size_t)(a.channels * type_size(a.param_type)), st);
    }
    return launched(name);
}

} // namespace

} // namespace ffcvb

using namespace ffcvb;

extern "C" int ffcvb_group_norm(const ffcvb_group_norm_args *args, void *workspace, void *stream) { return call(args, workspace, stream, false); }
extern "C" int ffcvb_group_norm_backward(const ffcvb_group_norm_args *args, void *workspace, void *stream) { return call(args, workspace, stream, true); }
extern "C" int64_t ffcvb_group_norm_workspace(const ffcvb_group_norm_args *args, int backward) {
    return !args || wrong(*args, backward != 0) || args->samples == 0 || args->positions == 0 ? 0 : plan_of(*args, backward != 0).bytes;
}
