// Cross entropy against labels, mixed labels or probabilities, with its gradient (sm_100a).
//
// With T the target's probabilities, S their sum and lse = log sum exp x, a row's loss is S * lse - sum T x and
// its gradient S * exp(x - lse) - T.  A warp takes a row of up to 1024 logits, a CTA one of up to 56 KB, a cluster a longer one.  Every
// thread copies its part of the row into shared memory, in places of its own; a pass over it keeps the largest logit so far and the
// sum of exponentials relative to that (in 32 bits), which are joined over the row's threads; a second pass makes the gradient.  So
// the row crosses HBM once each way, and several CTAs per SM load, compute and store at different times.
#include "training.h"
#include "two.h"

namespace ffcvb {

namespace {

// (Differences are taken before the factor: a row masked with the type's lowest value has no product with it.)
constexpr float kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float exp2_of(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float exp_of(float x) { return exp2_of(x * kLog2e); }

// What a row's target is besides probabilities per class: at most two classes with their weights, and the same
// `flat` for all.
struct Picks {
    long long label[2];
    float weight[2];
    float flat;
    float total;  // S
    bool ignored, bad;
};

__device__ __forceinline__ Picks picks_of(const ffcvb_cross_entropy_args &a, long long row) {
    Picks p{{-1, -1}, {0.0f, 0.0f}, a.smoothing / (float)a.classes, 0.0f, false, false};
    const float sure = 1.0f - a.smoothing;
    if (a.target_kind == FFCVB_TARGET_LABELS) {
        p.label[0] = static_cast<const int64_t *>(a.target)[row * a.target_stride];
        p.weight[0] = sure;
        p.ignored = a.has_ignore && p.label[0] == a.ignore_index;
        p.bad = p.label[0] < 0 || p.label[0] >= a.classes;
        p.total = sure + a.smoothing;
    } else if (a.target_kind == FFCVB_TARGET_MIXED) {
        const float *m = static_cast<const float *>(a.target) + row * a.target_stride;
        const float l0 = m[0], l1 = m[1], lam = m[2];
        p.bad = !(l0 >= 0.0f && l0 < (float)a.classes && l1 >= 0.0f && l1 < (float)a.classes);
        if (!p.bad) {
            p.label[0] = (long long)l0;
            p.label[1] = (long long)l1;
        }
        p.weight[0] = sure * lam;
        p.weight[1] = sure * (1.0f - lam);
        p.total = p.weight[0] + p.weight[1] + a.smoothing;
    }
    return p;
}

// N probabilities from place `at` on, those of classes [from, to) of the pack; 0 for the others.
template <int N>
__device__ __forceinline__ void probabilities(float (&p)[N], const ffcvb_cross_entropy_args &a, long long at, int from, int to, bool wide) {
    if (N > 1 && wide && a.target_type == FFCVB_TYPE_F32) {
#pragma unroll
        for (int j = 0; j < N; j += 4) {
            float4 f = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (j < to && j + 4 > from) f = *reinterpret_cast<const float4 *>(static_cast<const float *>(a.target) + at + j);
            p[j] = f.x, p[j + 1] = f.y, p[j + 2] = f.z, p[j + 3] = f.w;
        }
#pragma unroll
        for (int j = 0; j < N; j++)
            if (j < from || j >= to) p[j] = 0.0f;
        return;
    }
#pragma unroll
    for (int j = 0; j < N; j++) {
        p[j] = 0.0f;
        if (j < from || j >= to) continue;
        if (a.target_type == FFCVB_TYPE_F32)
            p[j] = static_cast<const float *>(a.target)[at + j];
        else if (a.target_type == FFCVB_TYPE_F16)
            p[j] = to_float(static_cast<const __half *>(a.target)[at + j]);
        else
            p[j] = to_float(static_cast<const __nv_bfloat16 *>(a.target)[at + j]);
    }
}

__device__ __forceinline__ void copy16(uint32_t to, const void *from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}

// The largest logit of a row and the sum of exponentials relative to it, and what else is summed up.
struct Found {
    float top, sum, dot, mass;
    // joins two parts of a row
    __device__ __forceinline__ void join(float t, float s, float d, float m) {
        const float most = fmaxf(top, t);
        // (nothing but what is no number is added to a part without a maximum)
        sum = (top == -INFINITY ? sum : sum * exp_of(top - most)) + (t == -INFINITY ? s : s * exp_of(t - most));
        top = most;
        dot += d;
        mass += m;
    }
    template <bool MORE> __device__ __forceinline__ void join_warp() {
        float most = warp_max(top);
        sum = warp_sum(top == -INFINITY ? sum : sum * exp_of(top - most));
        top = most;
        if (MORE) {
            dot = warp_sum(dot);
            mass = warp_sum(mass);
        }
    }
};

// How rows are dealt out: packs of a CTA's part of a row; whether parts are copied to shared memory; whether probabilities can be read
// 16 bytes at a time.
struct Deal {
    int part, staged, soft_wide;
};

// WIDE: 16 bytes at a time from the 16-byte boundary at or before the row on (what lies before the row there is left out); logits and
// gradient then lie alike to these boundaries.  WARP: a row per warp, four warps per CTA.
template <typename T, bool WIDE, bool SOFT, bool WARP>
__global__ void __launch_bounds__(WARP ? 128 : 512)
rows_kernel(const __grid_constant__ ffcvb_cross_entropy_args a, const Deal deal) {
    constexpr int N = WIDE ? kWide<T> : 1;
    __shared__ float4 s_part[16];
    __shared__ float4 s_there[8]; // from the cluster's CTAs
    extern __shared__ uint4 s_row[];
    uint32_t rank = 0, ranks = 1;
    if (!WARP) {
        asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
        asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
        if (ranks > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); // (this one has begun)
    }
    const int thread = WARP ? threadIdx.x & 31 : threadIdx.x, threads = WARP ? 32 : blockDim.x;
    const long long row = WARP ? blockIdx.x * 4ll + (threadIdx.x >> 5) : blockIdx.x / ranks;
    if (WARP && row >= a.rows) return;
    const int classes = (int)a.classes;
    const T *x = static_cast<const T *>(a.logits) + row * a.logits_stride;
    T *g = a.grad ? static_cast<T *>(a.grad) + row * a.grad_stride : nullptr;
    const int lead = WIDE ? (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T)) : 0;
    const int packs = (lead + classes + N - 1) / N;
    // this CTA's packs, [first, last); the row's first and last are not wholly of the row
    const int first = (int)rank * deal.part, last = min(packs, first + deal.part);
    const int head = lead > 0 ? 0 : -1, tail = (lead + classes) % N ? packs - 1 : -1;
    const T *x0 = x - lead;
    const uint32_t mine = (uint32_t)__cvta_generic_to_shared(s_row + (WARP ? (threadIdx.x >> 5) * deal.part : 0) + thread);
    const bool staged = WIDE && deal.staged && !a.from_stats;
    if (staged) {
        uint32_t to = mine;
        for (int k = first + thread; k < last; k += threads, to += threads * 16) copy16(to, x0 + (long long)k * N);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    const Picks p = picks_of(a, row);
    if (p.ignored || p.bad) { // (all of a cluster's CTAs alike)
        if (ranks > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
        const float v = p.ignored ? 0.0f : NAN;
        if (g)
            for (long long c = (long long)first * N - lead + thread; c < (long long)last * N - lead && c < classes; c += threads)
                if (c >= 0) g[c] = from_float<T>(v);
        if (thread == 0 && rank == 0 && !a.from_stats) {
            a.row_loss[row] = v;
            if (a.stats) reinterpret_cast<float2 *>(a.stats)[row] = make_float2(v, v);
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        return;
    }
    const long long soft_row = row * a.target_stride - lead;
    const float sure = 1.0f - a.smoothing;
    float picked = 0.0f; // of the labels' logits
    if (!SOFT && thread == 0 && rank == 0 && !a.from_stats) {
#pragma unroll
        for (int k = 0; k < 2; k++)
            if (p.weight[k] != 0.0f) picked += p.weight[k] * to_float(x[p.label[k]]);
    }
    // classes [from, to) of pack k are the row's
    auto ends = [&](int k, int &from, int &to) {
        from = k == head ? lead : 0;
        to = k == tail ? lead + classes - k * N : N;
    };
    auto fetch = [&](Pack<T, N> &pack, int k, uint32_t from) {
        if (staged) {
            if constexpr (WIDE)
                asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(pack.raw.x), "=r"(pack.raw.y), "=r"(pack.raw.z), "=r"(pack.raw.w) : "r"(from) : "memory");
        } else {
            pack.load(x0 + (long long)k * N);
        }
    };
    if (ranks > 1 && a.from_stats) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    float row_top, over, total = p.total; // (over: 1 / sum of exp(x - row_top), 0 where there is nothing)
    if (!a.from_stats) {
        Found f{-INFINITY, 0.0f, 0.0f, 0.0f};
        float base = 0.0f; // top, where there is one
        if (staged) asm volatile("cp.async.wait_group 0;" ::: "memory");
        uint32_t at = mine;
#pragma unroll 2
        for (int k = first + thread; k < last; k += threads, at += threads * 16) {
            Pack<T, N> pack;
            fetch(pack, k, at);
            float v[N];
            pack.get(v);
            if (WIDE && (k == head || k == tail)) {
                int from, to;
                ends(k, from, to);
#pragma unroll
                for (int j = 0; j < N; j++)
                    if (j < from || j >= to) v[j] = -INFINITY;
            }
            if (SOFT) {
                int from, to;
                ends(k, from, to);
                float t[N];
                probabilities<N>(t, a, soft_row + (long long)k * N, from, to, deal.soft_wide);
#pragma unroll
                for (int j = 0; j < N; j++) {
                    t[j] = j >= from && j < to ? sure * t[j] + p.flat : 0.0f;
                    f.mass += t[j];
                    if (t[j] > 0.0f) f.dot += t[j] * v[j];
                }
            } else if (p.flat > 0.0f) {
                int from, to;
                ends(k, from, to);
                float part = 0.0f;
#pragma unroll
                for (int j = 0; j < N; j++) part += j >= from && j < to ? v[j] : 0.0f;
                f.dot += p.flat * part;
            }
            float most = v[0];
#pragma unroll
            for (int j = 1; j < N; j++) most = fmaxf(most, v[j]);
            if (most > f.top) {
                if (f.top != -INFINITY) f.sum *= exp_of(f.top - most);
                f.top = base = most;
            }
            if constexpr (N == 1) {
                f.sum += exp_of(v[0] - base);
            } else {
                Two part(0.0f, 0.0f);
                const Two minus(-base, -base), log2e(kLog2e, kLog2e);
#pragma unroll
                for (int j = 0; j < N; j += 2) {
                    const Two d = mul_rn(add_rn(Two(v[j], v[j + 1]), minus), log2e);
                    part = add_rn(part, Two(exp2_of(d.lo()), exp2_of(d.hi())));
                }
                f.sum += part.lo() + part.hi();
            }
        }
        f.dot += picked;
        f.join_warp<true>();
        if (!WARP) {
            const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
            if (lane == 0) s_part[threadIdx.x >> 5] = make_float4(f.top, f.sum, f.dot, f.mass);
            __syncthreads();
            const float4 other = lane < warps ? s_part[lane] : make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
            f = Found{other.x, other.y, other.z, other.w};
            f.join_warp<true>();
            if (ranks > 1) {
                asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); // all have begun
                if (threadIdx.x < ranks) {
                    uint32_t there;
                    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"((uint32_t)__cvta_generic_to_shared(s_there + rank)), "r"(threadIdx.x));
                    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(there), "f"(f.top), "f"(f.sum), "f"(f.dot), "f"(f.mass) : "memory");
                }
                asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
                f = Found{s_there[0].x, s_there[0].y, s_there[0].z, s_there[0].w};
                for (uint32_t k = 1; k < ranks; k++) f.join(s_there[k].x, s_there[k].y, s_there[k].z, s_there[k].w);
            }
        }
        row_top = f.top == -INFINITY ? 0.0f : f.top;
        over = f.sum == 0.0f ? 0.0f : 1.0f / f.sum;
        if (SOFT) total = f.mass;
        if (thread == 0 && rank == 0) {
            a.row_loss[row] = f.sum == 0.0f ? 0.0f : total * (row_top + logf(f.sum)) - f.dot;
            if (a.stats) reinterpret_cast<float2 *>(a.stats)[row] = make_float2(row_top, over);
        }
    } else {
        const float2 stats = reinterpret_cast<const float2 *>(a.stats)[row];
        row_top = stats.x;
        over = stats.y;
        if (SOFT) { // the whole row's, by every CTA of a cluster
            float mass = 0.0f;
            for (int k = thread; k < packs; k += threads) {
                int from, to;
                ends(k, from, to);
                float t[N];
                probabilities<N>(t, a, soft_row + (long long)k * N, from, to, deal.soft_wide);
#pragma unroll
                for (int j = 0; j < N; j++) mass += j >= from && j < to ? sure * t[j] + p.flat : 0.0f;
            }
            mass = warp_sum(mass);
            if (!WARP) {
                const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
                if (lane == 0) s_part[threadIdx.x >> 5].x = mass;
                __syncthreads();
                mass = warp_sum(lane < warps ? s_part[lane].x : 0.0f);
            }
            total = mass;
        }
    }
    if (!g) return;
    float k_row = a.scale;
    if (a.upstream) k_row *= a.upstream[a.upstream_per_row ? row : 0];
    if (a.mean) k_row /= a.has_ignore ? fmaxf(a.counted[0], 1.0f) : (float)a.rows;
    if (over == 0.0f) k_row = 0.0f;
    const float factor = k_row * total * over, flat = k_row * p.flat;
    T *g0 = g - lead;
    // packs of the labels
    const int at0 = p.label[0] < 0 ? -1 : ((int)p.label[0] + lead) / N, at1 = p.label[1] < 0 ? -1 : ((int)p.label[1] + lead) / N;
    uint32_t at = mine;
#pragma unroll 2
    for (int k = first + thread; k < last; k += threads, at += threads * 16) {
        Pack<T, N> pack;
        fetch(pack, k, at);
        float v[N];
        pack.get(v);
        if constexpr (N == 1) {
            v[0] = factor * exp_of(v[0] - row_top) - flat;
        } else {
            const Two minus(-row_top, -row_top), log2e(kLog2e, kLog2e), less(-flat, -flat), times(factor, factor);
#pragma unroll
            for (int j = 0; j < N; j += 2) {
                const Two d = mul_rn(add_rn(Two(v[j], v[j + 1]), minus), log2e);
                const Two e = fma_rn(Two(exp2_of(d.lo()), exp2_of(d.hi())), times, less);
                v[j] = e.lo();
                v[j + 1] = e.hi();
            }
        }
        if (SOFT) {
            int from, to;
            ends(k, from, to);
            float t[N];
            probabilities<N>(t, a, soft_row + (long long)k * N, from, to, deal.soft_wide);
#pragma unroll
            for (int j = 0; j < N; j++) v[j] -= k_row * sure * t[j];
        } else if (k == at0 || k == at1) {
#pragma unroll
            for (int j = 0; j < N; j++) {
                const int c = k * N + j - lead;
                if (c == (int)p.label[0]) v[j] -= k_row * p.weight[0];
                if (c == (int)p.label[1]) v[j] -= k_row * p.weight[1];
            }
        }
        pack.set(v);
        if (!WIDE || (k != head && k != tail)) {
            pack.store_once(g0 + (long long)k * N);
        } else {
            int from, to;
            ends(k, from, to);
#pragma unroll
            for (int j = 0; j < N; j++)
                if (j >= from && j < to) g0[(long long)k * N + j] = from_float<T>(v[j]);
        }
    }
}

// Rows whose label is not ignore_index.
__global__ void __launch_bounds__(1024)
count_kernel(const int64_t *__restrict__ labels, long long rows, long long stride, long long ignore, float *counted) {
    __shared__ int s_count[32];
    int n = 0;
    for (long long i = threadIdx.x; i < rows; i += 1024) n += labels[i * stride] != ignore;
    n = __reduce_add_sync(0xffffffffu, n);
    if ((threadIdx.x & 31) == 0) s_count[threadIdx.x >> 5] = n;
    __syncthreads();
    if (threadIdx.x < 32) {
        n = __reduce_add_sync(0xffffffffu, s_count[threadIdx.x]);
        if (threadIdx.x == 0) *counted = (float)n;
    }
}

// The rows' losses added up, always in the same order.
__global__ void __launch_bounds__(1024)
mean_kernel(const float *__restrict__ row_loss, long long rows, const float *counted, int mean, float *loss) {
    __shared__ double s_sum[32];
    double sum = 0.0;
    for (long long i = threadIdx.x; i < rows; i += 1024) sum += row_loss[i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if ((threadIdx.x & 31) == 0) s_sum[threadIdx.x >> 5] = sum;
    __syncthreads();
    if (threadIdx.x < 32) {
        sum = s_sum[threadIdx.x];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (threadIdx.x == 0) *loss = (float)(mean ? sum / (counted ? fmax((double)*counted, 1.0) : (double)rows) : sum);
    }
}

constexpr long long kPartBytes = 56 * 1024; // of a row in a CTA's shared memory: four CTAs per SM
constexpr long long kWarpClasses = 1024;    // of a row that a warp takes

template <typename T>
void launch_rows(const ffcvb_cross_entropy_args &a, cudaStream_t stream) {
    constexpr int W = 16 / (int)sizeof(T);
    const uintptr_t apart = reinterpret_cast<uintptr_t>(a.logits) ^ reinterpret_cast<uintptr_t>(a.grad);
    const bool wide = !a.grad || ((apart & 15) == 0 && (a.logits_stride - a.grad_stride) * (long long)sizeof(T) % 16 == 0);
    const bool soft = a.target_kind == FFCVB_TARGET_SOFT;
    const long long packs = wide ? (a.classes + W - 1) / W + 1 : a.classes; // (at most one more than without a lead)
    Deal deal{};
    deal.staged = wide && a.grad && !a.from_stats;
    // probabilities lie to 16-byte boundaries as the logits' packs do: same stride, both begin on one
    deal.soft_wide = soft && ((reinterpret_cast<uintptr_t>(a.logits) | reinterpret_cast<uintptr_t>(a.target)) & 15) == 0 &&
                     (a.logits_stride - a.target_stride) % W == 0;
    cudaLaunchConfig_t how{};
    cudaLaunchAttribute cluster{};
    how.stream = stream;
    auto run = [&](auto kernel) {
        if (how.dynamicSmemBytes > 40 * 1024) cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)how.dynamicSmemBytes);
        cudaLaunchKernelEx(&how, kernel, a, deal);
    };
    if (a.classes <= kWarpClasses) {
        deal.part = (int)packs;
        how.gridDim = dim3((unsigned)((a.rows + 3) / 4));
        how.blockDim = dim3(128);
        how.dynamicSmemBytes = deal.staged ? 4 * packs * 16 : 0;
        if (wide)
            run(soft ? rows_kernel<T, true, true, true> : rows_kernel<T, true, false, true>);
        else
            run(soft ? rows_kernel<T, false, true, true> : rows_kernel<T, false, false, true>);
        return;
    }
    // CTAs per row: until a part fits, and until there are two CTAs per SM (with few rows) of parts that are worth it
    int ctas = 1;
    while (ctas < 8 && ((deal.staged && (packs + ctas - 1) / ctas * 16 > kPartBytes) || (a.rows * ctas * 2 <= 2 * kSms && packs > 2048 * ctas))) ctas *= 2;
    deal.part = (int)((packs + ctas - 1) / ctas);
    if (deal.staged && deal.part * 16ll > kPartBytes) deal.staged = 0; // (then the second pass reads what the caches still have)
    const int threads = (deal.part / 8 + 31) / 32 * 32;
    how.gridDim = dim3((unsigned)(a.rows * ctas));
    how.blockDim = dim3(threads < 64 ? 64 : threads > 320 ? 320 : threads);
    how.dynamicSmemBytes = deal.staged ? deal.part * 16ll : 0;
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim.x = ctas;
    cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
    how.attrs = &cluster;
    how.numAttrs = ctas > 1;
    if (wide)
        run(soft ? rows_kernel<T, true, true, false> : rows_kernel<T, true, false, false>);
    else
        run(soft ? rows_kernel<T, false, true, false> : rows_kernel<T, false, false, false>);
}

} // namespace

} // namespace ffcvb

using namespace ffcvb;

extern "C" int ffcvb_cross_entropy(const ffcvb_cross_entropy_args *args, void *stream) {
    if (!args) return training_fail(FFCVB_E_ARG, "ffcvb_cross_entropy: no arguments");
    const ffcvb_cross_entropy_args &a = *args;
    if (a.rows < 0 || a.classes < 1 || a.rows > 0x0fffffff || a.classes > 0x7fffff00 || (a.type != FFCVB_TYPE_F32 && a.type != FFCVB_TYPE_F16 && a.type != FFCVB_TYPE_BF16))
        return training_fail(FFCVB_E_ARG, "ffcvb_cross_entropy: bad size or type");
    const bool needs_count = a.has_ignore && a.mean && a.target_kind == FFCVB_TARGET_LABELS;
    if (a.target_kind < FFCVB_TARGET_LABELS || a.target_kind > FFCVB_TARGET_SOFT || !(a.smoothing >= 0.0f && a.smoothing <= 1.0f) ||
        (a.rows > 0 && (!a.logits || !a.target || (a.from_stats ? !a.stats || !a.grad : !a.row_loss))) || (needs_count && !a.counted) ||
        (a.has_ignore && a.target_kind != FFCVB_TARGET_LABELS))
        return training_fail(FFCVB_E_ARG, "ffcvb_cross_entropy: bad argument");
    OnDevice here(a.device);
    if (!here.ok()) return training_fail(FFCVB_E_NODEVICE, "ffcvb_cross_entropy: no device %d", a.device);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (needs_count) count_kernel<<<1, 1024, 0, st>>>(static_cast<const int64_t *>(a.target), a.rows, a.target_stride, a.ignore_index, a.counted);
    if (a.rows > 0) with_type(a.type, [&](auto zero) { launch_rows<decltype(zero)>(a, st); });
    if (a.loss && !a.from_stats) mean_kernel<<<1, 1024, 0, st>>>(a.row_loss, a.rows, needs_count ? a.counted : nullptr, a.mean, a.loss);
    return launched("ffcvb_cross_entropy");
}
