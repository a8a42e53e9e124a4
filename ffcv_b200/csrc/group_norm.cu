// Group norm with an activation, of images that lie channels last, forward and backward (sm_100a).
//
// A group of a sample are its m = positions * channels / groups values.  With their mean and r = 1 / sqrt(var + eps), hat = (x - mean) r,
//   a = hat w + b,  y = act(a);  backward  da = dy act'(a),  dx = r (da w - mean(da w) - hat mean(da w hat)),  dw = sum da hat,  db = sum da.
// The means over a group are sums over its channels of w times the sums over positions of da and da hat, which the weights' gradients need too.
//
// What fits is held: some groups of a sample (channels of 64 bytes or more), at all positions, in the shared memory of a CTA or of a cluster's, so that x
// (backward x and dy) is read once.  Threads copy what they use themselves, in places of their own, and exchange moments or sums
// across the CTA and the cluster.  What does not fit is read twice, by kernels for the sums, for joining them, and for the values.
//
// What bounds it: instructions, for the activation above all.  256 x 56 x 56 x 256 bf16 values with SiLU take 172 us forward and 321 backward, 125 and 188 at the rate of a copy: about 15 and 28
// instructions for a value, of which half the turns to issue are used, and the unit for exponentials and reciprocals 50 % of the time; the rest waits for copies and for the group's last value.  What is read twice is bound by HBM:
// 4 x 512 x 512 x 128 forward 159 us, 123 at the rate of a copy.  2 x 7 x 7 x 512 take 11 us for both directions: three launches.
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

// (What is held, by CTAs of 128: 56 x 56 x 256 forward and backward 187 and 385 us, 250 and 449 by CTAs of 256, which wait for more of their own.)
constexpr int kThreads = 256, kHeldThreads = 128;
constexpr int kAhead = 6;       // packs of x that a thread has on their way a second time
constexpr int kMostGroups = 32; // of a CTA
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float exp2_of(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float inverse_of(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ Two all(float v) { return Two(v, v); }

// 1 / (1 + exp(-a))
__device__ __forceinline__ Two gate_of(Two a) {
    const Two t = mul_rn(a, all(-kLog2e)), e = add_rn(Two(exp2_of(t.lo()), exp2_of(t.hi())), all(1.0f));
    return Two(inverse_of(e.lo()), inverse_of(e.hi()));
}
// The normal distribution's density at a, and its integral up to a.  With z = |a| / sqrt(2) and t = 1 / (1 + 0.42 z) the integral up to -|a| is
// t P(t) exp(-z^2) / 2; P is a polynomial fitted to that for z up to 6, to 3.3e-8 of the value.
__device__ __forceinline__ void normal(Two a, Two &density, Two &integral) {
    const Two u = fma_rn(Two(fabsf(a.lo()), fabsf(a.hi())), all(0.42f * 0.70710678118654752f), all(1.0f));
    const Two t(inverse_of(u.lo()), inverse_of(u.hi()));
    const Two square = mul_rn(mul_rn(a, a), all(-0.5f * kLog2e)), e(exp2_of(square.lo()), exp2_of(square.hi()));
    Two p = fma_rn(all(0.5f * 0.076194151358683f), t, all(0.5f * -0.3458746854890851f));
    p = fma_rn(p, t, all(0.5f * 0.4864512135112419f));
    p = fma_rn(p, t, all(0.5f * -0.174528421558005f));
    p = fma_rn(p, t, all(0.5f * 0.2932564906472867f));
    p = fma_rn(p, t, all(0.5f * 0.18682665698819034f));
    p = fma_rn(p, t, all(0.5f * 0.24094708374661222f));
    p = fma_rn(p, t, all(0.5f * 0.23672753345776956f));
    const Two tail = mul_rn(mul_rn(p, t), e), rest = sub_rn(all(1.0f), tail);
    integral = Two(a.lo() > 0.0f ? rest.lo() : tail.lo(), a.hi() > 0.0f ? rest.hi() : tail.hi());
    density = mul_rn(e, all(0.39894228040143268f));
}

// act(a), in pairs
template <int P> __device__ __forceinline__ void activate(Two (&v)[P], int kind) {
    if (kind == FFCVB_ACT_SILU) {
#pragma unroll
        for (int i = 0; i < P; i++) v[i] = mul_rn(v[i], gate_of(v[i]));
    } else if (kind == FFCVB_ACT_GELU) {
#pragma unroll
        for (int i = 0; i < P; i++) {
            Two density, integral;
            normal(v[i], density, integral);
            v[i] = mul_rn(v[i], integral);
        }
    } else if (kind == FFCVB_ACT_RELU) { // (NaN stays)
#pragma unroll
        for (int i = 0; i < P; i++) v[i] = Two(v[i].lo() < 0.0f ? 0.0f : v[i].lo(), v[i].hi() < 0.0f ? 0.0f : v[i].hi());
    }
}
// act'(a) dy in the place of dy
template <int P> __device__ __forceinline__ void slope(Two (&d)[P], const Two (&a)[P], int kind) {
    if (kind == FFCVB_ACT_SILU) {
#pragma unroll
        for (int i = 0; i < P; i++) {
            const Two gate = gate_of(a[i]), rest = sub_rn(all(1.0f), gate);
            d[i] = mul_rn(mul_rn(d[i], gate), fma_rn(a[i], rest, all(1.0f)));
        }
    } else if (kind == FFCVB_ACT_GELU) {
#pragma unroll
        for (int i = 0; i < P; i++) {
            Two density, integral;
            normal(a[i], density, integral);
            d[i] = mul_rn(d[i], fma_rn(a[i], density, integral));
        }
    } else if (kind == FFCVB_ACT_RELU) {
#pragma unroll
        for (int i = 0; i < P; i++) d[i] = Two(a[i].lo() > 0.0f ? d[i].lo() : 0.0f, a[i].hi() > 0.0f ? d[i].hi() : 0.0f);
    }
}

// A pack's values in pairs; the one pair of a single value has a 0 beside it.
template <int W> constexpr int kPairs = (W + 1) / 2;
template <typename T, int W> __device__ __forceinline__ void get_pairs(Two (&v)[kPairs<W>], const Pack<T, W> &pack) {
    float f[W];
    pack.get(f);
#pragma unroll
    for (int i = 0; i < kPairs<W>; i++) v[i] = Two(f[2 * i], W == 1 ? 0.0f : f[(2 * i + 1) % W]);
}
template <typename T, int W> __device__ __forceinline__ void put_pairs(T *to, const Two (&v)[kPairs<W>]) {
    float f[W];
#pragma unroll
    for (int j = 0; j < W; j++) f[j] = v[j / 2].half(j & 1);
    Pack<T, W> pack;
    pack.set(f);
    pack.store(to);
}

// Which groups a pack's channels are of: `left` those before `split`, the next one the others (SPLIT; else all are of one).
struct Groups {
    int left, split;
    // (the channel's middle over `per`: exact for as many channels as there may be)
    __device__ __forceinline__ Groups(int pack, int w, int per) : left((int)(((float)(pack * w) + 0.5f) / (float)per)), split(min(w, (left + 1) * per - pack * w)) {}
};
// A number of a pack's groups for each of its channels.
template <int W, bool SPLIT> struct Each {
    Two v[SPLIT ? kPairs<W> : 1];
    __device__ __forceinline__ void set(float left, float right, int split) {
#pragma unroll
        for (int i = 0; i < (SPLIT ? kPairs<W> : 1); i++) v[i] = Two(!SPLIT || 2 * i < split ? left : right, !SPLIT || 2 * i + 1 < split ? left : right);
    }
    __device__ __forceinline__ Two operator[](int i) const { return v[SPLIT ? i : 0]; }
};

// How many, their mean, and the sum of squares around it.
struct Moments {
    float n, mean, squares;
    __device__ __forceinline__ void join(Moments o) {
        const float both = n + o.n, share = __fdividef(o.n, fmaxf(both, 1.0f)), apart = o.mean - mean, step = apart * share;
        squares += fmaf(apart * step, n, o.squares);
        mean += step;
        n = both;
    }
    // of groups of LANES lanes; the lowest has the result
    template <int LANES = 32> __device__ __forceinline__ void join_lanes() {
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1)
            join(Moments{__shfl_down_sync(0xffffffffu, n, o), __shfl_down_sync(0xffffffffu, mean, o), __shfl_down_sync(0xffffffffu, squares, o)});
    }
    __device__ __forceinline__ float rate(float eps) const { return rsqrtf(squares / n + eps); }
};

// A thread's values of W channels, added up relative to a pivot for each group.  With the mean of some of the values as the pivot, m of the n that are
// added up, its square's distance from their mean is at most n / m variances, and the variance has so many roundings of 2^-24 of error at most: n / m is a
// thread's number of positions here.
template <int W, bool SPLIT> struct Collected {
    static constexpr int P = kPairs<W>;
    Each<W, SPLIT> pivot;
    Two sum[P], squares[P];
    __device__ __forceinline__ Collected() {
#pragma unroll
        for (int i = 0; i < P; i++) sum[i] = squares[i] = all(0.0f);
    }
    __device__ __forceinline__ void add(const Two (&v)[P]) {
#pragma unroll
        for (int i = 0; i < P; i++) {
            const Two d = sub_rn(v[i], pivot[i]);
            sum[i] = add_rn(sum[i], d);
            squares[i] = fma_rn(d, d, squares[i]);
        }
    }
    // Sums of the channels before `split`, or of those from it on.
    static __device__ __forceinline__ float of(const Two (&v)[P], int split, bool right) {
        if constexpr (!SPLIT) {
            Two s = v[0];
#pragma unroll
            for (int i = 1; i < P; i++) s = add_rn(s, v[i]);
            return W == 1 ? s.lo() : s.lo() + s.hi();
        }
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < W; j++) s += (j < split) != right ? v[j / 2].half(j & 1) : 0.0f;
        return s;
    }
};
// What is left of sums of n values around a pivot.
__device__ __forceinline__ Moments moments_of(float n, float pivot, float sum, float squares) {
    const float away = __fdividef(sum, fmaxf(n, 1.0f)), around = squares - sum * away;
    return Moments{n, pivot + away, around < 0.0f ? 0.0f : around}; // (NaN stays)
}

// W neighbouring parameters in pairs, or what stands for them.
__device__ __forceinline__ float parameter(const void *from, int type, long long c, float other) {
    return !from                    ? other
           : type == FFCVB_TYPE_F32 ? static_cast<const float *>(from)[c]
           : type == FFCVB_TYPE_F16 ? to_float(static_cast<const __half *>(from)[c])
                                    : to_float(static_cast<const __nv_bfloat16 *>(from)[c]);
}
template <int W> __device__ __forceinline__ void parameters(Two (&v)[kPairs<W>], const void *from, int type, long long c, float other) {
    float f[W];
    auto of = [&](auto *at) {
        using T = std::remove_const_t<std::remove_pointer_t<decltype(at)>>;
        if constexpr (W * sizeof(T) <= 16) {
            if (reinterpret_cast<uintptr_t>(at) % 16 == 0) { // (c is a multiple of W)
                Pack<T, W> pack;
                pack.load(at + c);
                pack.get(f);
                return;
            }
        }
#pragma unroll
        for (int j = 0; j < W; j++) f[j] = to_float(at[c + j]);
    };
    if (!from) {
#pragma unroll
        for (int j = 0; j < W; j++) f[j] = other;
    } else if (type == FFCVB_TYPE_F32) {
        of(static_cast<const float *>(from));
    } else if (type == FFCVB_TYPE_F16) {
        of(static_cast<const __half *>(from));
    } else {
        of(static_cast<const __nv_bfloat16 *>(from));
    }
#pragma unroll
    for (int i = 0; i < kPairs<W>; i++) v[i] = Two(f[2 * i], W == 1 ? 0.0f : f[(2 * i + 1) % W]);
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

__device__ __forceinline__ void cluster_begun() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() { asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void store_there(const void *mine, uint32_t rank, float v) {
    uint32_t at;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(mine)), "r"(rank));
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at), "f"(v) : "memory");
}

// ---- held: a CTA or a cluster has some groups of a sample at all positions ---------------------------------------------

// Groups of a CTA, packs of a position in them, of which `lanes` positions at once; positions of a CTA; CTAs of a cluster; channels of a group.
struct Deal {
    int groups, packs, lanes, rows, ctas, per;
};
// Of a CTA: its cluster's rank, first group and sample; its thread's row and pack.
struct Held {
    int rank, group0, row, pack, first, last;
    long long sample;
    __device__ __forceinline__ Held(const Deal &deal, int positions) {
        rank = blockIdx.x & (deal.ctas - 1); // (1, 2, 4 or 8)
        group0 = (blockIdx.x >> (31 - __clz(deal.ctas))) * deal.groups;
        sample = blockIdx.y;
        row = (int)(((float)threadIdx.x + 0.5f) / (float)deal.packs);
        pack = threadIdx.x - row * deal.packs;
        first = rank * deal.rows;
        last = min(first + deal.rows, positions);
    }
};
// Lanes of a warp that have the same pack of a power of two of them can be joined; then a warp has one row of partial results, else each row has.
__host__ __device__ constexpr bool joined(int packs) { return packs <= 32 && (packs & (packs - 1)) == 0; }
__host__ __device__ constexpr int part_rows(int packs, int lanes, int threads) { return joined(packs) ? threads / 32 : lanes; }

// s_moments[side][row][pack]: of a CTA's packs, from all its rows.
template <typename T, int W, bool SPLIT>
__global__ void __launch_bounds__(kHeldThreads) held_forward_kernel(const __grid_constant__ ffcvb_group_norm_args a, const Deal deal) {
    constexpr int P = kPairs<W>, SIDES = SPLIT ? 2 : 1, N = kHeldThreads;
    __shared__ Moments s_moments[SIDES][N];
    __shared__ Moments s_there[8][kMostGroups]; // of the cluster's CTAs
    __shared__ float2 s_stats[kMostGroups];
    extern __shared__ uint4 s_held[];
    wait_for_previous();
    let_next_begin();
    if (deal.ctas > 1) cluster_begun();
    const Held me(deal, (int)a.positions);
    const Groups groups(me.pack, W, deal.per);
    const int channel = me.group0 * deal.per + me.pack * W;
    const bool used = me.row < deal.lanes;
    Pack<T, W> *held = reinterpret_cast<Pack<T, W> *>(s_held) + threadIdx.x;
    if (used) {
        const T *from = static_cast<const T *>(a.x) + me.sample * a.x_sample + (me.first + me.row) * a.x_position + channel;
        const long long step = deal.lanes * a.x_position;
        Pack<T, W> *to = held;
        for (int r = me.first + me.row; r < me.last; r += deal.lanes, to += N, from += step) copy_pack(to, from);
    }
    Two w[P], b[P];
    if (used) {
        parameters<W>(w, a.weight, a.param_type, channel, 1.0f);
        parameters<W>(b, a.bias, a.param_type, channel, 0.0f);
    }
    copies_done();
    {
        Collected<W, SPLIT> values;
        const int turns = used && me.first + me.row < me.last ? (me.last - me.first - me.row - 1) / deal.lanes + 1 : 0;
        // the pivots: means of the thread's first values; of those of the warp's lanes with the same pack, where they are joined
        const float there[2] = {SPLIT ? (float)groups.split : (float)W, (float)(W - groups.split)};
        float pivot[2] = {0.0f, 0.0f}, n[2];
        if (turns) {
            Two v[P];
            get_pairs<T, W>(v, *held);
#pragma unroll
            for (int side = 0; side < SIDES; side++) pivot[side] = values.of(v, groups.split, side);
        }
#pragma unroll
        for (int side = 0; side < SIDES; side++) {
            float m = turns ? there[side] : 0.0f;
            n[side] = (float)turns * there[side];
            if (joined(deal.packs))
                for (int o = 16; o >= deal.packs; o >>= 1) {
                    pivot[side] += __shfl_xor_sync(0xffffffffu, pivot[side], o);
                    m += __shfl_xor_sync(0xffffffffu, m, o);
                    n[side] += __shfl_xor_sync(0xffffffffu, n[side], o);
                }
            pivot[side] = __fdividef(pivot[side], fmaxf(m, 1.0f));
        }
        values.pivot.set(pivot[0], pivot[SIDES - 1], groups.split);
        const Pack<T, W> *from = held;
#pragma unroll 2
        for (int k = 0; k < turns; k++, from += N) {
            Two v[P];
            get_pairs<T, W>(v, *from);
            values.add(v);
        }
#pragma unroll
        for (int side = 0; side < SIDES; side++) {
            float sum = values.of(values.sum, groups.split, side), squares = values.of(values.squares, groups.split, side);
            int at = threadIdx.x; // (row by row)
            bool writes = used;
            if (joined(deal.packs)) {
                for (int o = 16; o >= deal.packs; o >>= 1) {
                    sum += __shfl_xor_sync(0xffffffffu, sum, o);
                    squares += __shfl_xor_sync(0xffffffffu, squares, o);
                }
                at = (threadIdx.x >> 5) * deal.packs + (threadIdx.x & 31);
                writes = (threadIdx.x & 31) < deal.packs;
            }
            if (writes) s_moments[side][at] = moments_of(n[side], pivot[side], sum, squares);
        }
    }
    __syncthreads();
    if (deal.ctas > 1) cluster_wait(); // all have begun
    // a quarter of a warp has a group: its packs, in all rows of partial results
    const int rows = part_rows(deal.packs, deal.lanes, N);
    for (int g0 = threadIdx.x >> 5 << 2; g0 < deal.groups; g0 += N / 8) {
        const int g = g0 + (threadIdx.x & 31) / 8, e0 = threadIdx.x & 7;
        Moments found{0.0f, 0.0f, 0.0f};
        if (g < deal.groups) {
            const int pack0 = g * deal.per / W, each = ((g + 1) * deal.per - 1) / W - pack0 + 1;
            for (int k = pack0; k < pack0 + each; k++) {
                const int side = SPLIT && Groups(k, W, deal.per).left != g;
                for (int r = e0; r < rows; r += 8) found.join(s_moments[side][r * deal.packs + k]);
            }
        }
        found.join_lanes<8>();
        found.n = __shfl_sync(0xffffffffu, found.n, threadIdx.x & 24);
        found.mean = __shfl_sync(0xffffffffu, found.mean, threadIdx.x & 24);
        found.squares = __shfl_sync(0xffffffffu, found.squares, threadIdx.x & 24);
        if (g < deal.groups && e0 < deal.ctas) {
            Moments *to = &s_there[me.rank][g];
            if (deal.ctas == 1) {
                *to = found;
            } else {
                store_there(&to->n, e0, found.n);
                store_there(&to->mean, e0, found.mean);
                store_there(&to->squares, e0, found.squares);
            }
        }
    }
    if (deal.ctas > 1)
        cluster_sync();
    else
        __syncthreads();
    if (threadIdx.x < deal.groups) {
        Moments whole = s_there[0][threadIdx.x];
        for (int k = 1; k < deal.ctas; k++) whole.join(s_there[k][threadIdx.x]);
        const float2 stats = make_float2(whole.mean, whole.rate(a.eps));
        s_stats[threadIdx.x] = stats;
        if (me.rank == 0) reinterpret_cast<float2 *>(a.stats)[me.sample * a.groups + me.group0 + threadIdx.x] = stats;
    }
    __syncthreads();
    if (!used) return;
    const float2 left = s_stats[groups.left], right = SPLIT ? s_stats[min(groups.left + 1, deal.groups - 1)] : left;
    Each<W, SPLIT> less, rates;
    less.set(left.x, right.x, groups.split);
    rates.set(left.y, right.y, groups.split);
#pragma unroll
    for (int i = 0; i < P; i++) w[i] = mul_rn(w[i], rates[i]);
    T *to = static_cast<T *>(a.y) + (me.sample * a.positions + me.first + me.row) * a.channels + channel;
    const long long step = deal.lanes * a.channels;
    const Pack<T, W> *from = held;
#pragma unroll 2
    for (int r = me.first + me.row; r < me.last; r += deal.lanes, from += N, to += step) {
        Two v[P];
        get_pairs<T, W>(v, *from);
#pragma unroll
        for (int i = 0; i < P; i++) v[i] = fma_rn(sub_rn(v[i], less[i]), w[i], b[i]);
        activate(v, a.activation);
        put_pairs<T, W>(to, v);
    }
}

// A thread's sums over its positions of da and of da hat, of W channels.
template <int W> struct Sums {
    static constexpr int P = kPairs<W>;
    Two da[P], hat[P];
    __device__ __forceinline__ Sums() {
#pragma unroll
        for (int i = 0; i < P; i++) da[i] = hat[i] = all(0.0f);
    }
    __device__ __forceinline__ void add(const Two (&h)[P], const Two (&d)[P]) {
#pragma unroll
        for (int i = 0; i < P; i++) {
            da[i] = add_rn(da[i], d[i]);
            hat[i] = fma_rn(d[i], h[i], hat[i]);
        }
    }
    // (from sums of da c)
    template <bool SPLIT> __device__ __forceinline__ void times(const Each<W, SPLIT> &rate) {
#pragma unroll
        for (int i = 0; i < P; i++) hat[i] = mul_rn(hat[i], rate[i]);
    }
    __device__ __forceinline__ float2 of(int j) const { return make_float2(da[j / 2].half(j & 1), hat[j / 2].half(j & 1)); }
    // Lanes of a warp that have the same pack, `packs` (a power of two) apart: the lowest has the sum.
    __device__ __forceinline__ void join_lanes(int packs) {
        for (int o = 16; o >= packs; o >>= 1)
#pragma unroll
            for (int i = 0; i < P; i++) {
                da[i] = add_rn(da[i], Two(__shfl_down_sync(0xffffffffu, da[i].lo(), o), __shfl_down_sync(0xffffffffu, da[i].hi(), o)));
                hat[i] = add_rn(hat[i], Two(__shfl_down_sync(0xffffffffu, hat[i].lo(), o), __shfl_down_sync(0xffffffffu, hat[i].hi(), o)));
            }
    }
};

// Sums of a CTA's threads joined over its positions: s_sums[channel]; `s_all` is room for part_rows() times the channels.
template <int W> __device__ __forceinline__ void channel_sums(Sums<W> &mine, bool used, int row, int pack, int lanes, int packs, float2 *s_all, float2 *s_sums) {
    const int channels = packs * W, rows = part_rows(packs, lanes, kHeldThreads);
    bool writes = used;
    if (joined(packs)) {
        mine.join_lanes(packs);
        row = threadIdx.x >> 5;
        writes = (threadIdx.x & 31) < packs;
    }
    if (writes)
#pragma unroll
        for (int j = 0; j < W; j++) s_all[row * channels + pack * W + j] = mine.of(j);
    __syncthreads();
    // rows are halved until at most four are left, always in the same order
    int n = rows;
    while (n > 4) {
        const int half = (n + 1) / 2;
        for (int i = threadIdx.x; i < (n - half) * channels; i += kHeldThreads) {
            s_all[i].x += s_all[i + half * channels].x;
            s_all[i].y += s_all[i + half * channels].y;
        }
        n = half;
        __syncthreads();
    }
    for (int i = threadIdx.x; i < channels; i += kHeldThreads) {
        float2 sum = s_all[i];
        for (int k = 1; k < n; k++) {
            sum.x += s_all[k * channels + i].x;
            sum.y += s_all[k * channels + i].y;
        }
        s_sums[i] = sum;
    }
}

// What a thread needs for da of W channels, with c = x - mean: a = c (w r) + b; and for dx = w r da - r mean(da w) - c r^2 mean(da w hat).
template <typename T, int W, bool SPLIT> struct Back {
    static constexpr int P = kPairs<W>;
    Two w[P], b[P]; // (w r)
    Each<W, SPLIT> mean, rate;
    int kind;
    __device__ __forceinline__ Back() {}
    __device__ __forceinline__ Back(const ffcvb_group_norm_args &a, long long sample, int channel, int group, const Groups &groups) : kind(a.activation) {
        parameters<W>(w, a.weight, a.param_type, channel, 1.0f);
        parameters<W>(b, a.bias, a.param_type, channel, 0.0f);
        const float2 *stats = reinterpret_cast<const float2 *>(a.stats) + sample * a.groups;
        const float2 left = stats[group], right = SPLIT ? stats[min(group + 1, (int)a.groups - 1)] : left;
        mean.set(left.x, right.x, groups.split);
        rate.set(left.y, right.y, groups.split);
#pragma unroll
        for (int i = 0; i < P; i++) w[i] = mul_rn(w[i], rate[i]);
    }
    // c
    __device__ __forceinline__ void center(const Pack<T, W> &x, Two (&c)[P]) const {
        get_pairs<T, W>(c, x);
#pragma unroll
        for (int i = 0; i < P; i++) c[i] = sub_rn(c[i], mean[i]);
    }
    // c and a
    __device__ __forceinline__ void row(const Pack<T, W> &x, Two (&c)[P], Two (&v)[P]) const {
        get_pairs<T, W>(c, x);
#pragma unroll
        for (int i = 0; i < P; i++) {
            c[i] = sub_rn(c[i], mean[i]);
            v[i] = fma_rn(c[i], w[i], b[i]);
        }
    }
    // c and da
    __device__ __forceinline__ void row(const Pack<T, W> &x, const Pack<T, W> &dy, Two (&c)[P], Two (&da)[P]) const {
        Two v[P];
        row(x, c, v);
        get_pairs<T, W>(da, dy);
        slope(da, v, kind);
    }
    // `less`: r mean(da w) and -r^2 mean(da w hat)
    __device__ __forceinline__ void gradient(const Two (&c)[P], Two (&da)[P], const Each<W, SPLIT> &less, const Each<W, SPLIT> &less_c) const {
#pragma unroll
        for (int i = 0; i < P; i++) da[i] = fma_rn(c[i], less_c[i], fma_rn(da[i], w[i], less[i]));
    }
    // those from the groups' means
    __device__ __forceinline__ void means(Each<W, SPLIT> &less, Each<W, SPLIT> &less_c, float2 left, float2 right, int split) const {
        less.set(left.x, right.x, split);
        less_c.set(left.y, right.y, split);
#pragma unroll
        for (int i = 0; i < (SPLIT ? P : 1); i++) {
            const Two r = mul_rn(rate.v[i], all(-1.0f));
            less.v[i] = mul_rn(less.v[i], r);
            less_c.v[i] = mul_rn(mul_rn(less_c.v[i], r), rate.v[i]);
        }
    }
};

// da in 32 bits in the place of a pack of x and one of dy; in the place of dy alone, where that has as many bits.
template <typename T, int W> __device__ __forceinline__ void keep_pairs(Pack<T, W> *x, Pack<T, W> *dy, const Two (&v)[kPairs<W>]) {
    if constexpr (sizeof(T) == 4) {
        put_pairs<T, W>(reinterpret_cast<T *>(dy), v);
    } else if constexpr (W > 1) {
        float f[W];
#pragma unroll
        for (int i = 0; i < W; i++) f[i] = v[i / 2].half(i & 1);
        Pack<float, W / 2> half;
        half.set(reinterpret_cast<float(&)[W / 2]>(f[0]));
        half.store(reinterpret_cast<float *>(x));
        half.set(reinterpret_cast<float(&)[W / 2]>(f[W / 2]));
        half.store(reinterpret_cast<float *>(dy));
    }
}
template <typename T, int W> __device__ __forceinline__ void kept_pairs(Two (&v)[kPairs<W>], const Pack<T, W> *x, const Pack<T, W> *dy) {
    if constexpr (sizeof(T) == 4) {
        get_pairs<T, W>(v, *dy);
    } else if constexpr (W > 1) {
        float f[W];
        reinterpret_cast<const Pack<float, W / 2> *>(x)->get(reinterpret_cast<float(&)[W / 2]>(f[0]));
        reinterpret_cast<const Pack<float, W / 2> *>(dy)->get(reinterpret_cast<float(&)[W / 2]>(f[W / 2]));
#pragma unroll
        for (int i = 0; i < W / 2; i++) v[i] = Two(f[2 * i], f[2 * i + 1]);
    }
}

// room: (part_rows() + CTAs of the cluster) times the channels, of two floats; then, for each turn of the threads, x and dy
// Behind SiLU and GELU da stays for the second pass, in 32 bits where x and dy were, and of 16 bits x is read once more, out of L2, ahead of its use: backward 56 x 56 x 256 321 us,
// 359 where da is computed twice, 520 where it has room of its own beside x and dy, which other CTAs need; with 2, 4 and 8 packs ahead 332, 329 and 322 (28 x 28 x 512
// 174 with 6, 177 with 8).
template <typename T, int W, bool SPLIT>
__global__ void __launch_bounds__(kHeldThreads) held_backward_kernel(const __grid_constant__ ffcvb_group_norm_args a, const Deal deal, float2 *sums) {
    constexpr int P = kPairs<W>, N = kHeldThreads;
    __shared__ float2 s_group[kMostGroups];
    extern __shared__ uint4 s_held[];
    wait_for_previous();
    let_next_begin();
    if (deal.ctas > 1) cluster_begun();
    const Held me(deal, (int)a.positions);
    const int channels = deal.packs * W, rows = part_rows(deal.packs, deal.lanes, kHeldThreads);
    const Groups groups(me.pack, W, deal.per);
    const int channel = me.group0 * deal.per + me.pack * W;
    const bool used = me.row < deal.lanes;
    float2 *s_all = reinterpret_cast<float2 *>(s_held), *s_there = s_all + rows * channels; // [ctas][channels]
    Pack<T, W> *held = reinterpret_cast<Pack<T, W> *>(s_held + ((rows + deal.ctas) * channels + 1) / 2) + threadIdx.x;
    if (used) {
        const T *x = static_cast<const T *>(a.x) + me.sample * a.x_sample + (me.first + me.row) * a.x_position + channel;
        const T *dy = static_cast<const T *>(a.dy) + me.sample * a.dy_sample + (me.first + me.row) * a.dy_position + channel;
        const long long x_step = deal.lanes * a.x_position, dy_step = deal.lanes * a.dy_position;
        Pack<T, W> *to = held;
        for (int r = me.first + me.row; r < me.last; r += deal.lanes, to += 2 * N, x += x_step, dy += dy_step) {
            copy_pack(to, x);
            copy_pack(to + N, dy);
        }
    }
    Back<T, W, SPLIT> back;
    if (used) back = Back<T, W, SPLIT>(a, me.sample, channel, me.group0 + groups.left, groups);
    copies_done();
    const bool keep = (sizeof(T) == 4 || W > 1) && (a.activation == FFCVB_ACT_SILU || a.activation == FFCVB_ACT_GELU);
    {
        Sums<W> mine;
        if (used) {
            Pack<T, W> *from = held;
#pragma unroll 2
            for (int r = me.first + me.row; r < me.last; r += deal.lanes, from += 2 * N) {
                Two c[P], da[P];
                back.row(from[0], from[N], c, da);
                mine.add(c, da);
                if (keep) keep_pairs<T, W>(from, from + N, da);
            }
            mine.times(back.rate);
        }
        channel_sums<W>(mine, used, me.row, me.pack, deal.lanes, deal.packs, s_all, s_there + me.rank * channels);
    }
    // (x's values of the first turns once more)
    const T *again = static_cast<const T *>(a.x) + me.sample * a.x_sample + (me.first + me.row) * a.x_position + channel;
    const long long again_step = deal.lanes * a.x_position;
    Pack<T, W> ahead[kAhead];
    if (sizeof(T) == 2 && keep && used)
#pragma unroll
        for (int j = 0; j < kAhead; j++)
            if (me.first + me.row + j * deal.lanes < me.last) ahead[j].load(again + j * again_step);
    __syncthreads();
    if (deal.ctas > 1) {
        cluster_wait(); // all have begun
        for (int i = threadIdx.x; i < channels; i += kHeldThreads) {
            float2 *at = s_there + me.rank * channels + i;
            const float2 v = *at;
            for (int to = 0; to < deal.ctas; to++) {
                if (to == me.rank) continue;
                store_there(&at->x, to, v.x);
                store_there(&at->y, to, v.y);
            }
        }
        cluster_sync();
        for (int i = threadIdx.x; i < channels; i += kHeldThreads) {
            float2 whole = s_there[i];
            for (int k = 1; k < deal.ctas; k++) {
                whole.x += s_there[k * channels + i].x;
                whole.y += s_there[k * channels + i].y;
            }
            s_all[i] = whole;
        }
        __syncthreads();
    } else {
        s_all = s_there;
    }
    if (me.rank == 0)
        for (int i = threadIdx.x; i < channels; i += kHeldThreads) sums[me.sample * a.channels + me.group0 * deal.per + i] = s_all[i];
    for (int g = threadIdx.x >> 5; g < deal.groups; g += kHeldThreads / 32) {
        float2 mean = make_float2(0.0f, 0.0f);
        for (int c = threadIdx.x & 31; c < deal.per; c += 32) {
            const float one = parameter(a.weight, a.param_type, me.group0 * deal.per + g * deal.per + c, 1.0f);
            mean.x = fmaf(one, s_all[g * deal.per + c].x, mean.x);
            mean.y = fmaf(one, s_all[g * deal.per + c].y, mean.y);
        }
        const float over = 1.0f / ((float)a.positions * (float)deal.per);
        mean.x = warp_sum(mean.x) * over;
        mean.y = warp_sum(mean.y) * over;
        if ((threadIdx.x & 31) == 0) s_group[g] = mean;
    }
    __syncthreads();
    if (!used || !a.dx) return;
    Each<W, SPLIT> less, less_c;
    back.means(less, less_c, s_group[groups.left], s_group[min(groups.left + 1, deal.groups - 1)], groups.split);
    T *to = static_cast<T *>(a.dx) + (me.sample * a.positions + me.first + me.row) * a.channels + channel;
    const long long step = deal.lanes * a.channels;
    const Pack<T, W> *from = held;
    if (sizeof(T) == 2 && keep) {
        again += kAhead * again_step;
#pragma unroll 1
        for (int r = me.first + me.row; r < me.last; r += kAhead * deal.lanes) {
#pragma unroll
            for (int j = 0; j < kAhead; j++) {
                if (r + j * deal.lanes >= me.last) break;
                Two c[P], da[P];
                back.center(ahead[j], c);
                if (r + (j + kAhead) * deal.lanes < me.last) ahead[j].load(again);
                kept_pairs<T, W>(da, from, from + N);
                back.gradient(c, da, less, less_c);
                put_pairs<T, W>(to, da);
                from += 2 * N, to += step, again += again_step;
            }
        }
        return;
    }
#pragma unroll 2
    for (int r = me.first + me.row; r < me.last; r += deal.lanes, from += 2 * N, to += step) {
        Two c[P], da[P];
        if (sizeof(T) == 4 && keep) {
            back.center(from[0], c);
            kept_pairs<T, W>(da, from, from + N);
        } else {
            back.row(from[0], from[N], c, da);
        }
        back.gradient(c, da, less, less_c);
        put_pairs<T, W>(to, da);
    }
}

// ---- not held: sums of slabs of positions, joined; then the values -------------------------------------------------------
//
// All samples' slabs in one launch, the values' from the last one back: 4 x 512 x 512 x 128 forward 236 us as built first, 298 to 336 in launches over as many samples as L2 holds,
// which end and begin too often.  Three CTAs on an SM of the two kernels that read x and dy: backward 431 us, 507 with the registers that the compiler chooses.

// Packs of a position, of which a CTA has `columns`, and `lanes` positions at once; positions of a slab, and slabs.
struct Slabs {
    int packs, columns, lanes, rows, slabs;
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
    p.sample = n / s.slabs;
    p.first = p.slab * s.rows;
    p.last = min(p.first + s.rows, positions);
    p.used = p.row < s.lanes && p.pack < s.packs;
    return p;
}

// Calls f(pack of x, pack of dy, position) for a thread's positions, four of them loaded before the first is used (two with dy).
template <typename T, int W, bool TWO, typename F>
__device__ __forceinline__ void each_position(const Place &p, int lanes, const T *x, long long x_step, const T *dy, long long dy_step, F &&f) {
    constexpr int BATCH = TWO ? 2 : 4;
    int r = p.first + p.row;
    x += r * x_step;
    dy += r * dy_step;
    for (; r + (BATCH - 1) * lanes < p.last; r += BATCH * lanes) {
        Pack<T, W> one[BATCH], other[BATCH];
#pragma unroll
        for (int i = 0; i < BATCH; i++, x += lanes * x_step, dy += lanes * dy_step) {
            one[i].load(x);
            if (TWO) other[i].load(dy);
        }
#pragma unroll
        for (int i = 0; i < BATCH; i++) f(one[i], other[i], r + i * lanes);
    }
    for (; r < p.last; r += lanes, x += lanes * x_step, dy += lanes * dy_step) {
        Pack<T, W> one, other;
        one.load(x);
        if (TWO) other.load(dy);
        f(one, other, r);
    }
}

// parts: [samples][slabs][packs][sides], mean and squares around it
template <typename T, int W, bool SPLIT>
__global__ void __launch_bounds__(kThreads) moments_kernel(const __grid_constant__ ffcvb_group_norm_args a, const Slabs s, float2 *parts) {
    constexpr int P = kPairs<W>, SIDES = SPLIT ? 2 : 1;
    __shared__ Moments s_moments[SIDES][kThreads];
    wait_for_previous();
    let_next_begin();
    const Place p = place_of(s, (int)a.positions, false);
    const Groups groups(p.pack, W, (int)(a.channels / a.groups));
    Collected<W, SPLIT> values;
    float pivot[2] = {0.0f, 0.0f}, n[2] = {0.0f, 0.0f};
    if (p.used && p.first + p.row < p.last) {
        const T *x = static_cast<const T *>(a.x) + p.sample * a.x_sample + p.pack * W;
        const float turns = (float)((p.last - p.first - p.row - 1) / s.lanes + 1);
        Pack<T, W> pack;
        Two v[P];
        pack.load(x + (p.first + p.row) * a.x_position);
        get_pairs<T, W>(v, pack);
#pragma unroll
        for (int side = 0; side < SIDES; side++) {
            const float there = !SPLIT ? (float)W : side ? (float)(W - groups.split) : (float)groups.split;
            pivot[side] = __fdividef(values.of(v, groups.split, side), fmaxf(there, 1.0f));
            n[side] = turns * there;
        }
        values.pivot.set(pivot[0], pivot[SIDES - 1], groups.split);
        each_position<T, W, false>(p, s.lanes, x, a.x_position, x, 0, [&](const Pack<T, W> &pack, const Pack<T, W> &, int) {
            Two v[P];
            get_pairs<T, W>(v, pack);
            values.add(v);
        });
    }
#pragma unroll
    for (int side = 0; side < SIDES; side++)
        s_moments[side][threadIdx.x] = moments_of(n[side], pivot[side], values.of(values.sum, groups.split, side), values.of(values.squares, groups.split, side));
    __syncthreads();
    for (int i = threadIdx.x; i < s.columns * SIDES; i += kThreads) {
        const int column = i % s.columns, side = i / s.columns, pack = blockIdx.y * s.columns + column;
        if (pack >= s.packs) continue;
        Moments whole = s_moments[side][column];
        for (int k = 1; k < s.lanes; k++) whole.join(s_moments[side][k * s.columns + column]);
        parts[((p.sample * s.slabs + p.slab) * s.packs + pack) * SIDES + side] = make_float2(whole.mean, whole.squares);
    }
}

// A CTA per group.
template <int W, bool SPLIT> __global__ void __launch_bounds__(kThreads) join_moments_kernel(const __grid_constant__ ffcvb_group_norm_args a, const Slabs s, const float2 *parts) {
    constexpr int SIDES = SPLIT ? 2 : 1;
    __shared__ Moments s_part[kThreads / 32];
    wait_for_previous();
    let_next_begin();
    const long long sample = blockIdx.x / a.groups;
    const int group = (int)(blockIdx.x % a.groups), per = (int)(a.channels / a.groups), pack0 = (int)((long long)group * per / W);
    const int each = (int)(((long long)(group + 1) * per - 1) / W) - pack0 + 1;
    Moments found{0.0f, 0.0f, 0.0f};
    for (long long e = threadIdx.x; e < (long long)s.slabs * each; e += kThreads) {
        const int slab = (int)(e / each), pack = pack0 + (int)(e % each);
        const Groups groups(pack, W, per);
        const int side = SPLIT && groups.left != group, there = !SPLIT ? W : side ? W - groups.split : groups.split;
        const float2 part = parts[((sample * s.slabs + slab) * s.packs + pack) * SIDES + side];
        found.join(Moments{(float)min(s.rows, (int)a.positions - slab * s.rows) * (float)there, part.x, part.y});
    }
    found.join_lanes();
    if ((threadIdx.x & 31) == 0) s_part[threadIdx.x >> 5] = found;
    __syncthreads();
    if (threadIdx.x) return;
    for (int k = 1; k < kThreads / 32; k++) found.join(s_part[k]);
    reinterpret_cast<float2 *>(a.stats)[sample * a.groups + group] = make_float2(found.mean, found.rate(a.eps));
}

template <typename T, int W, bool SPLIT>
__global__ void __launch_bounds__(kThreads) values_kernel(const __grid_constant__ ffcvb_group_norm_args a, const Slabs s) {
    constexpr int P = kPairs<W>;
    wait_for_previous();
    let_next_begin();
    const Place p = place_of(s, (int)a.positions, true);
    if (!p.used) return;
    const Groups groups(p.pack, W, (int)(a.channels / a.groups));
    const int channel = p.pack * W;
    const Back<T, W, SPLIT> by(a, p.sample, channel, groups.left, groups);
    const T *x = static_cast<const T *>(a.x) + p.sample * a.x_sample + channel;
    T *y = static_cast<T *>(a.y) + p.sample * a.positions * a.channels + channel;
    each_position<T, W, false>(p, s.lanes, x, a.x_position, x, 0, [&](const Pack<T, W> &pack, const Pack<T, W> &, int r) {
        Two c[P], v[P];
        by.row(pack, c, v);
        activate(v, a.activation);
        put_pairs<T, W>(y + r * a.channels, v);
    });
}

// parts: [samples][slabs][channels]
template <typename T, int W, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 3) sums_kernel(const __grid_constant__ ffcvb_group_norm_args a, const Slabs s, float2 *parts) {
    constexpr int P = kPairs<W>;
    __shared__ float2 s_all[kThreads * W];
    wait_for_previous();
    let_next_begin();
    const Place p = place_of(s, (int)a.positions, false);
    Sums<W> mine;
    if (p.used) {
        const Groups groups(p.pack, W, (int)(a.channels / a.groups));
        const int channel = p.pack * W;
        const Back<T, W, SPLIT> back(a, p.sample, channel, groups.left, groups);
        const T *x = static_cast<const T *>(a.x) + p.sample * a.x_sample + channel, *dy = static_cast<const T *>(a.dy) + p.sample * a.dy_sample + channel;
        each_position<T, W, true>(p, s.lanes, x, a.x_position, dy, a.dy_position, [&](const Pack<T, W> &one, const Pack<T, W> &other, int) {
            Two c[P], da[P];
            back.row(one, other, c, da);
            mine.add(c, da);
        });
        mine.times(back.rate);
    }
    float2 *to = parts + (p.sample * s.slabs + p.slab) * a.channels + blockIdx.y * s.columns * W;
    const int channels = s.columns * W, there = min(channels, (int)a.channels - (int)blockIdx.y * channels);
    if (p.row < s.lanes)
#pragma unroll
        for (int j = 0; j < W; j++) s_all[p.row * channels + threadIdx.x % s.columns * W + j] = mine.of(j);
    __syncthreads();
    for (int c = threadIdx.x; c < there; c += kThreads) {
        float2 whole = s_all[c];
        for (int k = 1; k < s.lanes; k++) {
            whole.x += s_all[k * channels + c].x;
            whole.y += s_all[k * channels + c].y;
        }
        to[c] = whole;
    }
}

// A CTA per group: its channels' sums, [samples][channels], and its means, [samples][groups].
__global__ void __launch_bounds__(kThreads) join_sums_kernel(const __grid_constant__ ffcvb_group_norm_args a, const Slabs s, const float2 *parts, float2 *sums, float2 *means) {
    __shared__ float2 s_part[kThreads / 32];
    wait_for_previous();
    let_next_begin();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, per = (int)(a.channels / a.groups), group = (int)(blockIdx.x % a.groups);
    const long long sample = blockIdx.x / a.groups;
    float2 mean = make_float2(0.0f, 0.0f);
    for (int c = group * per + warp; c < (group + 1) * per; c += kThreads / 32) {
        float2 whole = make_float2(0.0f, 0.0f);
#pragma unroll 4
        for (int k = lane; k < s.slabs; k += 32) {
            const float2 part = parts[(sample * s.slabs + k) * a.channels + c];
            whole.x += part.x;
            whole.y += part.y;
        }
        whole.x = warp_sum(whole.x);
        whole.y = warp_sum(whole.y);
        const float w = parameter(a.weight, a.param_type, c, 1.0f);
        mean.x = fmaf(w, whole.x, mean.x);
        mean.y = fmaf(w, whole.y, mean.y);
        if (lane == 0) sums[sample * a.channels + c] = whole;
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

template <typename T, int W, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 3) gradient_kernel(const __grid_constant__ ffcvb_group_norm_args a, const Slabs s, const float2 *means) {
    constexpr int P = kPairs<W>;
    wait_for_previous();
    let_next_begin();
    const Place p = place_of(s, (int)a.positions, true);
    if (!p.used) return;
    const Groups groups(p.pack, W, (int)(a.channels / a.groups));
    const int channel = p.pack * W;
    const Back<T, W, SPLIT> back(a, p.sample, channel, groups.left, groups);
    Each<W, SPLIT> less, less_c;
    back.means(less, less_c, means[p.sample * a.groups + groups.left], means[p.sample * a.groups + min(groups.left + 1, (int)a.groups - 1)], groups.split);
    const T *x = static_cast<const T *>(a.x) + p.sample * a.x_sample + channel, *dy = static_cast<const T *>(a.dy) + p.sample * a.dy_sample + channel;
    T *dx = static_cast<T *>(a.dx) + p.sample * a.positions * a.channels + channel;
    each_position<T, W, true>(p, s.lanes, x, a.x_position, dy, a.dy_position, [&](const Pack<T, W> &one, const Pack<T, W> &other, int r) {
        Two c[P], da[P];
        back.row(one, other, c, da);
        back.gradient(c, da, less, less_c);
        put_pairs<T, W>(dx + r * a.channels, da);
    });
}

// The parameters' gradients: samples' sums added up, 32 channels per CTA.
__global__ void __launch_bounds__(1024) samples_kernel(const __grid_constant__ ffcvb_group_norm_args a, const float2 *sums) {
    __shared__ float2 s_part[32][32];
    wait_for_previous();
    let_next_begin();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long c = blockIdx.x * 32ll + lane;
    float2 whole = make_float2(0.0f, 0.0f);
    if (c < a.channels)
#pragma unroll 4
        for (long long n = warp; n < a.samples; n += 32) {
            const float2 part = sums[n * a.channels + c];
            whole.x += part.x;
            whole.y += part.y;
        }
    s_part[warp][lane] = whole;
    __syncthreads();
    if (warp || c >= a.channels) return;
    for (int k = 1; k < 32; k++) {
        whole.x += s_part[k][lane].x;
        whole.y += s_part[k][lane].y;
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
    put(a.dbias, whole.x);
    put(a.dweight, whole.y);
}

// ---- the host's part -------------------------------------------------------------------------------------------------

// Bytes that a CTA holds at most; of one that is not alone rather so little that there are many on an SM, in clusters of up to eight.  (Forward and backward: 512 x 14 x 14 x 1024 84 and 134
// us, 84 and 161 with single CTAs of up to 51 KB; 1024 x 7 x 7 x 2048 88 and 167, 88 and 391; 256 x 56 x 56 x 256 with parts of 51 KB 180 and 321, of 36 172 and 321; up to 72 KB by themselves
// 206 forward.  Clusters of 16: 184 and 319, and 128 x 64 x 64 x 320, which is read twice, backward 538 where it takes 421.)
constexpr int64_t kMostHeld = 74 * 1024, kHeld = 36 * 1024;
// Bytes of neighbouring channels that a CTA reads at least, where there are as many; and what it holds rather of small images, as long as there are six CTAs for
// every SM.  (56 x 56 x 256 forward and backward 187 and 385 us, 223 and 477 with 32 bytes; small images: 14 x 14 x 1024 forward 87 us, 119 with 64 bytes, 7 x 7 x 2048 83 and 195.)
constexpr int64_t kNeighbours = 64, kSmall = 32 * 1024;
// Positions of a thread in a slab: as many as bring eight CTAs to every SM.  (Forward and backward: 1 x 256 x 256 x 64 13 and 23 us, 17 and 28 with one position at least; 2 x 64 x 64 x 320
// 12 and 23, 12 and 35; 4 x 512 x 512 x 128 159 and 307, 162 and 310 with 16 at most, 183 and 359 with 8.)
constexpr int64_t kLeastTurns = 4, kMostTurns = 64;

// Values of a pack: of one group or of two neighbouring ones (`split`), and where they begin as their size has it.
int width_of(const ffcvb_group_norm_args &a, bool backward) {
    const int size = type_size(a.type);
    int w = 16 / size;
    auto fits = [&](const void *p, int64_t sample, int64_t position) {
        return reinterpret_cast<uintptr_t>(p) % (w * size) == 0 && (a.samples <= 1 || sample % w == 0) && (a.positions <= 1 || position % w == 0);
    };
    const int64_t per = a.channels / a.groups;
    for (; w > 1; w /= 2)
        if (a.channels % w == 0 && (per >= w || w == 2 * per) && fits(a.x, a.x_sample, a.x_position) &&
            (backward ? fits(a.dy, a.dy_sample, a.dy_position) && (!a.dx || fits(a.dx, 0, 0)) : fits(a.y, 0, 0)))
            break;
    return w;
}

struct Plan {
    int width;
    bool split, held;
    Deal deal;
    int64_t room;     // bytes of shared memory
    Slabs slabs;
    int64_t parts, means, sums, bytes; // offsets in the workspace
};

Plan plan_of(const ffcvb_group_norm_args &a, bool backward) {
    Plan p{};
    const int size = type_size(a.type), w = p.width = width_of(a, backward);
    const int64_t per = a.channels / a.groups;
    p.split = per % w != 0;
    Deal &d = p.deal;
    d.groups = 1;
    while (d.groups * 2 <= kMostGroups && a.groups % (d.groups * 2) == 0 &&
           (d.groups * per * size < kNeighbours || d.groups * per % w != 0 ||
            (d.groups * 2 * per * size * a.positions <= kSmall && d.groups * 2 * per / w <= 64 && a.samples * a.groups / (d.groups * 2) >= kSms * 6)))
        d.groups *= 2;
    constexpr int threads = kHeldThreads;
    const int64_t packs = d.groups * per / w;
    if (packs <= threads && d.groups * per % w == 0 && a.samples <= 65535) {
        d.packs = (int)packs;
        d.per = (int)per;
        d.lanes = (int)std::min<int64_t>(threads / packs, std::max<int64_t>(a.positions, 1));
        auto room_of = [&](int ctas) {
            const int64_t rows = (a.positions + ctas - 1) / ctas, turns = (rows + d.lanes - 1) / d.lanes;
            return turns * threads * w * size * (backward ? 2 : 1) + (backward ? ((part_rows(d.packs, d.lanes, threads) + ctas) * packs * w + 1) / 2 * 16 : 0);
        };
        d.ctas = 1;
        if (room_of(1) > kMostHeld)
            while (d.ctas < 8 && room_of(d.ctas) > kHeld) d.ctas *= 2;
        p.room = room_of(d.ctas);
        p.held = p.room <= kMostHeld;
        d.rows = (int)((a.positions + d.ctas - 1) / d.ctas);
    }
    Slabs &s = p.slabs;
    s.packs = (int)(a.channels / w);
    s.columns = std::min(s.packs, kThreads);
    s.lanes = std::max(1, kThreads / s.columns);
    const int64_t ctas = a.samples * ((s.packs + s.columns - 1) / s.columns), fair = (a.positions * ctas + (int64_t)s.lanes * kSms * 8 - 1) / ((int64_t)s.lanes * kSms * 8);
    s.rows = (int)std::min<int64_t>(a.positions, std::clamp(fair, kLeastTurns, kMostTurns) * s.lanes);
    s.slabs = s.rows ? (int)((a.positions + s.rows - 1) / s.rows) : 0;
    int64_t at = 0;
    auto take = [&](bool wanted, int64_t bytes) {
        const int64_t here = at;
        if (wanted) at += (bytes + 255) / 256 * 256;
        return here;
    };
    p.parts = take(!p.held, a.samples * s.slabs * (backward ? a.channels : s.packs * (p.split ? 2 : 1)) * 8);
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
    if ((reinterpret_cast<uintptr_t>(a.stats) & 7) != 0) return "stats begin on 8 bytes";
    if (backward && !a.dx && !a.dweight && !a.dbias) return "nothing to do";
    if (a.samples > 0 && a.positions > 0 && a.samples * plan_of(a, backward).slabs.slabs > INT32_MAX) return "too many values";
    return nullptr;
}

// Calls f with a value of the type, the width of a call's packs, and whether they have two groups.
template <int W> using Width = std::integral_constant<int, W>;
template <typename T, typename F> void with_width(int w, bool split, F &&f) {
    auto with = [&](auto width) {
        if (split)
            f(T{}, width, std::true_type{});
        else
            f(T{}, width, std::false_type{});
    };
    if constexpr (sizeof(T) == 2)
        if (w == 8) return with(Width<8>{});
    if (w == 4) return with(Width<4>{});
    if (w == 2) return with(Width<2>{});
    f(T{}, Width<1>{}, std::false_type{});
}

template <typename... Params, typename... Given> void launch_cluster(void (*kernel)(Params...), dim3 grid, int threads, int cluster, int64_t room, cudaStream_t stream, Given &&...given) {
    cudaLaunchConfig_t how{};
    cudaLaunchAttribute with[2] = {};
    with[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    with[0].val.programmaticStreamSerializationAllowed = 1;
    with[1].id = cudaLaunchAttributeClusterDimension;
    with[1].val.clusterDim.x = cluster;
    with[1].val.clusterDim.y = with[1].val.clusterDim.z = 1;
    how.gridDim = grid;
    how.blockDim = dim3(threads);
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
        with_width<decltype(zero)>(p.width, p.split, [&](auto of, auto width, auto split) {
            using T = decltype(of);
            constexpr int W = decltype(width)::value;
            constexpr bool SPLIT = decltype(split)::value;
            if (p.held) {
                launch_cluster(held_forward_kernel<T, W, SPLIT>, dim3((unsigned)(a.groups / p.deal.groups * p.deal.ctas), (unsigned)a.samples), kHeldThreads, p.deal.ctas, p.room, st, a, p.deal);
                return;
            }
            float2 *parts = reinterpret_cast<float2 *>(room + p.parts);
            const Slabs &s = p.slabs;
            const dim3 grid((unsigned)(a.samples * s.slabs), (unsigned)((s.packs + s.columns - 1) / s.columns));
            launch_early(moments_kernel<T, W, SPLIT>, grid, kThreads, 0, st, a, s, parts);
            launch_early(join_moments_kernel<W, SPLIT>, (unsigned)(a.samples * a.groups), kThreads, 0, st, a, s, parts);
            launch_early(values_kernel<T, W, SPLIT>, grid, kThreads, 0, st, a, s);
        });
    });
}

void run_backward(const ffcvb_group_norm_args &a, uint8_t *room, cudaStream_t st) {
    const Plan p = plan_of(a, true);
    float2 *sums = reinterpret_cast<float2 *>(room + p.sums);
    with_type(a.type, [&](auto zero) {
        with_width<decltype(zero)>(p.width, p.split, [&](auto of, auto width, auto split) {
            using T = decltype(of);
            constexpr int W = decltype(width)::value;
            constexpr bool SPLIT = decltype(split)::value;
            if (p.held) {
                launch_cluster(held_backward_kernel<T, W, SPLIT>, dim3((unsigned)(a.groups / p.deal.groups * p.deal.ctas), (unsigned)a.samples), kHeldThreads, p.deal.ctas, p.room, st, a, p.deal, sums);
                return;
            }
            float2 *parts = reinterpret_cast<float2 *>(room + p.parts), *means = reinterpret_cast<float2 *>(room + p.means);
            const Slabs &s = p.slabs;
            const dim3 grid((unsigned)(a.samples * s.slabs), (unsigned)((s.packs + s.columns - 1) / s.columns));
            launch_early(sums_kernel<T, W, SPLIT>, grid, kThreads, 0, st, a, s, parts);
            launch_early(join_sums_kernel, (unsigned)(a.samples * a.groups), kThreads, 0, st, a, s, parts, sums, means);
            if (a.dx) launch_early(gradient_kernel<T, W, SPLIT>, grid, kThreads, 0, st, a, s, means);
        });
    });
    if (a.dweight || a.dbias) launch_early(samples_kernel, (unsigned)((a.channels + 31) / 32), 1024, 0, st, a, sums);
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
    } else if (!backward) { // (a mean of nothing is no number, and all bits of a NaN may be set)
        if (a.stats && a.samples > 0) cudaMemsetAsync(a.stats, 0xff, (size_t)(a.samples * a.groups * 8), st);
    } else {
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
