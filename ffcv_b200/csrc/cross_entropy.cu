// Cross entropy against labels, mixed labels or probabilities, with its gradient (sm_100a).
//
// With T the target's probabilities, S their sum and lse = log sum exp x, a row's loss is S * lse - sum T x and
// its gradient S * exp(x - lse) - T.  With the largest logit taken off, S * log sum exp(x - top) + sum T (top - x), the loss has terms of
// one sign alone, and no logit's size enters it.  Some lanes of a warp take a row of up to 8 KB, a CTA one of up to 56 KB, a cluster a longer one.  Every
// thread copies its part of the row into shared memory, in places of its own; a pass over it keeps the largest logit so far and the
// sum of exponentials relative to that (in 32 bits), which are joined over the row's threads; a second pass makes the gradient.  So
// the row crosses HBM once each way, and several CTAs per SM load, compute and store at different times.
//
// What bounds it: two exponentials per logit and the instructions around them; 8192 x 21841 bf16 logits take 129 us, 109 at the rate
// of a copy; with smoothing 130, with probabilities in 32 bits, which both passes read, 326.
#include "losses.h"

#include <type_traits>

namespace ffcvb {

namespace {

// N probabilities from class c of a row on.
template <int N>
__device__ __forceinline__ void probabilities(float (&p)[N], const ffcvb_cross_entropy_args &a, long long at, bool wide) {
    if (N > 1 && wide && a.target_type == FFCVB_TYPE_F32) {
#pragma unroll
        for (int j = 0; j < N; j += 4) {
            const float4 f = *reinterpret_cast<const float4 *>(static_cast<const float *>(a.target) + at + j);
            p[j] = f.x, p[j + 1] = f.y, p[j + 2] = f.z, p[j + 3] = f.w;
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < N; j++)
        p[j] = a.target_type == FFCVB_TYPE_F32   ? static_cast<const float *>(a.target)[at + j]
               : a.target_type == FFCVB_TYPE_F16 ? to_float(static_cast<const __half *>(a.target)[at + j])
                                                 : to_float(static_cast<const __nv_bfloat16 *>(a.target)[at + j]);
}

// The largest logit of a part of a row, at least kLowest, and the sum of exponentials relative to it; with targets besides labels also the
// sum of targets times logits, which are relative to it too, and the targets' sum.  (Where all logits are -inf the sum is 0: no difference
// here is that of two infinities of one sign, unless a logit is +inf.)  Relative sums stay finite where several logits are the type's
// lowest value, and keep the digits of logits that are all far from zero.
struct Found {
    float top, sum, dot, mass;
    // what a dot relative to `from` has more when it is relative to `to`, the larger (kept finite: there may be no mass yet)
    static __device__ __forceinline__ float shift(float mass, float from, float to) { return mass * fmaxf(from - to, kLowest); }
    __device__ __forceinline__ void join(float t, float s, float d, float m) {
        const float most = fmaxf(top, t);
        sum = sum * exp_of(top - most) + s * exp_of(t - most);
        dot = (dot + shift(mass, top, most)) + (d + shift(m, t, most));
        top = most;
        mass += m;
    }
    // joins those of groups of LANES lanes, in each of which all are in `mask`; `more`: dot and mass too
    template <int LANES> __device__ __forceinline__ void join_lanes(bool more, uint32_t mask) {
        float most = top;
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(mask, most, o));
        sum *= exp_of(top - most);
        if (more) dot += shift(mass, top, most);
        top = most;
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(mask, sum, o);
        if (!more) return;
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) dot += __shfl_xor_sync(mask, dot, o);
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) mass += __shfl_xor_sync(mask, mass, o);
    }
    template <int N> __device__ __forceinline__ void add(const float (&v)[N]) {
        float most = fmaxf(top, v[0]);
#pragma unroll
        for (int j = 1; j < N; j++) most = fmaxf(most, v[j]);
        sum *= exp_of(top - most);
        top = most;
        if constexpr (N == 1) {
            sum += exp_of(v[0] - top);
        } else {
            Two part[2] = {Two(0.0f, 0.0f), Two(0.0f, 0.0f)};
            const Two minus(-top, -top), log2e(kLog2e, kLog2e);
#pragma unroll
            for (int j = 0; j < N; j += 2) {
                const Two d = mul_rn(add_rn(Two(v[j], v[j + 1]), minus), log2e);
                part[j / 2 & 1] = add_rn(part[j / 2 & 1], Two(exp2_of(d.lo()), exp2_of(d.hi())));
            }
            part[0] = add_rn(part[0], part[1]);
            sum += part[0].lo() + part[0].hi();
        }
    }
};

// How rows are dealt out: whether logits and gradient lie alike to 16-byte boundaries; packs of a CTA's part of a row; whether
// probabilities can be read 16 bytes at a time.
struct Deal {
    int wide, part, soft_wide;
};

// A row's packs of 16 bytes are dealt out to its threads in turn; the few logits before and behind them (all, where logits and
// gradient lie differently to 16-byte boundaries) are taken one by one.  LANES: as many lanes of a warp (2 to 32) have a row, in CTAs of
// four warps; 0: a row per CTA or cluster.  STAGED: the packs go through shared memory; else they are read where they are needed.  (Ten CTAs per
// SM of lanes' rows: 16384 x 2000 bf16 with probabilities 56.4 us, 61.5 with the nine that the compiler's own choice of registers allows.)
template <typename T, bool STAGED, bool SOFT, int LANES>
__global__ void __launch_bounds__(LANES ? 128 : 256, LANES && STAGED ? 10 : 0)
rows_kernel(const __grid_constant__ ffcvb_cross_entropy_args a, const Deal deal) {
    constexpr bool WARP = LANES > 0;
    constexpr int N = kWide<T>, BATCH = STAGED ? 1 : 4; // packs that a thread has on their way
    __shared__ float4 s_part[8];
    __shared__ float4 s_there[8]; // from the cluster's CTAs
    extern __shared__ uint4 s_row[];
    wait_for_previous();
    let_next_begin();
    uint32_t rank = 0, ranks = 1;
    if (!WARP) {
        asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
        asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
        if (ranks > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); // (this one has begun)
    }
    const int thread = WARP ? threadIdx.x & (LANES - 1) : threadIdx.x, threads = WARP ? LANES : blockDim.x;
    const long long row = WARP ? blockIdx.x * (128ll / (WARP ? LANES : 1)) + threadIdx.x / (WARP ? LANES : 1) : blockIdx.x / ranks;
    const uint32_t mask = !WARP || LANES == 32 ? 0xffffffffu : ((1u << (LANES & 31)) - 1) << (threadIdx.x & 31 & -LANES); // lanes of the row
    if (WARP && row >= a.rows) return;
    const int classes = (int)a.classes;
    const T *x = static_cast<const T *>(a.logits) + row * a.logits_stride;
    T *g = a.grad ? static_cast<T *>(a.grad) + row * a.grad_stride : nullptr;
    // logits before the packs, packs of the row and of this CTA's part, logits besides packs
    const int lead = (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / (int)sizeof(T);
    const int before = deal.wide && lead < classes ? lead : classes;
    const int packs = (classes - before) / N, singles = classes - packs * N;
    const int first = (int)rank * deal.part, count = max(0, min(packs - first, deal.part));
    const T *x0 = x + before + (long long)first * N;
    const uint32_t mine = (uint32_t)__cvta_generic_to_shared(s_row + (WARP ? threadIdx.x / (WARP ? LANES : 1) * deal.part : 0) + thread);
    if (STAGED) {
        uint32_t to = mine;
        for (int k = thread; k < count; k += threads, to += threads * 16) copy16(to, x0 + (long long)k * N);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    auto single = [&](int k) { return k < before ? k : k + packs * N; }; // class of the k-th besides packs
    const Picks p = picks_of(a, row);
    if (p.ignored || p.bad) { // (all of a cluster's CTAs alike)
        const T v = from_float<T>(p.ignored ? 0.0f : NAN);
        if (g)
            for (int c = (int)rank * threads + thread; c < classes; c += (int)ranks * threads) g[c] = v;
        if (thread == 0 && rank == 0 && !a.from_stats) {
            a.row_loss[row] = to_float(v);
            if (a.stats) reinterpret_cast<float2 *>(a.stats)[row] = make_float2(to_float(v), to_float(v));
        }
        if (STAGED) asm volatile("cp.async.wait_group 0;" ::: "memory");
        if (ranks > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
        return;
    }
    const long long soft_row = row * a.target_stride;
    const float sure = 1.0f - a.smoothing;
    float picked[2] = {0.0f, 0.0f}; // the labels' logits
    if (!SOFT && thread == 0 && rank == 0 && !a.from_stats) {
#pragma unroll
        for (int k = 0; k < 2; k++)
            if (p.weight[k] != 0.0f) picked[k] = to_float(x[p.label[k]]);
    }
    // Calls f(values, class of the first) for this thread's packs: as many turns as all threads have, BATCH at a time, then what is left.
    const int turns = count / threads;
    auto each_pack = [&](auto &&f) {
        uint32_t at = mine;
        const T *from = x0 + (long long)thread * N;
        int c = before + (first + thread) * N;
        const int step = threads * N;
        auto load = [&](Pack<T, N> &pack, int i) {
            if constexpr (STAGED) {
                uint4 &r = pack.raw;
                asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(at + i * threads * 16) : "memory");
            } else {
                pack.load(from + (long long)i * step);
            }
        };
        auto work = [&](const Pack<T, N> &pack, int i) {
            float v[N];
            pack.get(v);
            f(v, c + i * step);
        };
        int k = 0;
        for (; k + BATCH <= turns; k += BATCH) {
            Pack<T, N> pack[BATCH];
#pragma unroll
            for (int i = 0; i < BATCH; i++) load(pack[i], i);
#pragma unroll
            for (int i = 0; i < BATCH; i++) work(pack[i], i);
            at += BATCH * threads * 16;
            from += (long long)BATCH * step;
            c += BATCH * step;
        }
        for (; k <= turns; k++) {
            if (k == turns && turns * threads + thread >= count) break;
            Pack<T, N> pack;
            load(pack, 0);
            work(pack, 0);
            at += threads * 16;
            from += step;
            c += step;
        }
    };
    auto each_single = [&](auto &&f) {
        for (int k = (int)rank * threads + thread; k < singles; k += (int)ranks * threads) f(single(k));
    };
    if (ranks > 1 && a.from_stats) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    float row_top, over, total = p.total; // (over: 1 / sum of exp(x - row_top), 0 where there is nothing)
    if (!a.from_stats) {
        Found f{kLowest, 0.0f, 0.0f, 0.0f};
        auto take = [&](auto &v, int c) {
            constexpr int M = sizeof(v) / 4;
            const float was = f.top;
            float t[M];
            if (SOFT) probabilities<M>(t, a, soft_row + c, deal.soft_wide);
            f.add(v);
            if (SOFT) {
                f.dot += Found::shift(f.mass, was, f.top);
                float part = 0.0f, mass = 0.0f;
#pragma unroll
                for (int j = 0; j < M; j++) {
                    t[j] = sure * t[j] + p.flat;
                    mass += t[j];
                    part += t[j] > 0.0f ? t[j] * (v[j] - f.top) : 0.0f;
                }
                f.dot += part;
                f.mass += mass;
            } else if (p.flat > 0.0f) {
                f.dot += Found::shift(f.mass, was, f.top);
                f.mass += M * p.flat;
                if constexpr (M == 1) {
                    f.dot += p.flat * (v[0] - f.top);
                } else { // (each times its target before they are added: the sum of two lowest values is none)
                    const Two minus(-f.top, -f.top), flat(p.flat, p.flat);
                    Two part(0.0f, 0.0f);
#pragma unroll
                    for (int j = 0; j < M; j += 2) part = fma_rn(add_rn(Two(v[j], v[j + 1]), minus), flat, part);
                    f.dot += part.lo() + part.hi();
                }
            }
        };
        each_single([&](int c) {
            const float v[1] = {to_float(x[c])};
            take(v, c);
        });
        if (STAGED) asm volatile("cp.async.wait_group 0;" ::: "memory");
        each_pack(take);
        const bool more = SOFT || p.flat > 0.0f;
        f.join_lanes<WARP ? LANES : 32>(more, mask);
        if (!WARP) {
            const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
            if (lane == 0) s_part[threadIdx.x >> 5] = make_float4(f.top, f.sum, f.dot, f.mass);
            __syncthreads();
            const float4 other = (lane & 7) < warps ? s_part[lane & 7] : make_float4(kLowest, 0.0f, 0.0f, 0.0f); // (at most eight)
            f = Found{other.x, other.y, other.z, other.w};
            f.join_lanes<8>(more, mask);
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
        row_top = f.top;
        over = f.sum == 0.0f ? 0.0f : 1.0f / f.sum;
        if (SOFT) total = f.mass;
        if (thread == 0 && rank == 0) {
#pragma unroll
            for (int k = 0; k < 2; k++)
                if (!SOFT && p.weight[k] != 0.0f) f.dot += p.weight[k] * (picked[k] - row_top);
            a.row_loss[row] = f.sum == 0.0f ? 0.0f : total * logf(f.sum) - f.dot;
            if (a.stats) reinterpret_cast<float2 *>(a.stats)[row] = make_float2(row_top, over);
        }
    } else {
        const float2 stats = reinterpret_cast<const float2 *>(a.stats)[row];
        row_top = stats.x;
        over = stats.y;
        if (SOFT) { // the whole row's, by every CTA of a cluster
            float mass = 0.0f;
            for (int c = thread; c < classes; c += threads) {
                float t[1];
                probabilities<1>(t, a, soft_row + c, false);
                mass += sure * t[0] + p.flat;
            }
#pragma unroll
            for (int o = WARP ? LANES / 2 : 16; o > 0; o >>= 1) mass += __shfl_xor_sync(mask, mass, o);
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
    each_single([&](int c) {
        float v = factor * exp_of(to_float(x[c]) - row_top) - flat;
        if (SOFT) {
            float t[1];
            probabilities<1>(t, a, soft_row + c, false);
            v -= k_row * sure * t[0];
        } else {
#pragma unroll
            for (int k = 0; k < 2; k++)
                if (c == (int)p.label[k]) v -= k_row * p.weight[k];
        }
        g[c] = from_float<T>(v);
    });
    const Two minus(-row_top, -row_top), log2e(kLog2e, kLog2e), less(-flat, -flat), times(factor, factor);
    each_pack([&](float(&v)[N], int c) {
#pragma unroll
        for (int j = 0; j < N; j += 2) {
            const Two d = mul_rn(add_rn(Two(v[j], v[j + 1]), minus), log2e);
            const Two e = fma_rn(Two(exp2_of(d.lo()), exp2_of(d.hi())), times, less);
            v[j] = e.lo();
            v[j + 1] = e.hi();
        }
        if (SOFT) {
            float t[N];
            probabilities<N>(t, a, soft_row + c, deal.soft_wide);
#pragma unroll
            for (int j = 0; j < N; j++) v[j] -= k_row * sure * t[j];
        }
        Pack<T, N> pack;
        pack.set(v);
        pack.store(g + c);
    });
    if (!SOFT) { // the labels' classes in packs: the thread that has just written them writes them again
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const int c = (int)p.label[k], in = c - before;
            if (c < 0 || in < 0 || in >= packs * N || in / N < first || (in / N - first) % threads != thread || in / N - first >= count) continue;
            float v = factor * exp_of(to_float(x[c]) - row_top) - flat - k_row * p.weight[k];
            if (p.label[0] == p.label[1]) v -= k_row * p.weight[k ^ 1];
            g[c] = from_float<T>(v);
        }
    }
}

// Rows whose label is not ignore_index.
__global__ void __launch_bounds__(1024)
count_kernel(const int64_t *__restrict__ labels, long long rows, long long stride, long long ignore, float *counted) {
    __shared__ int s_count[32];
    wait_for_previous();
    let_next_begin();
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
    wait_for_previous();
    double sum = 0.0;
#pragma unroll 8
    for (long long i = threadIdx.x; i < rows; i += 1024) sum += row_loss[i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if ((threadIdx.x & 31) == 0) s_sum[threadIdx.x >> 5] = sum;
    __syncthreads();
    if (threadIdx.x < 32) {
        sum = s_sum[threadIdx.x];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (threadIdx.x == 0) *loss = (float)(mean ? sum / fmax(counted ? (double)*counted : (double)rows, 1.0) : sum);
    }
}

// Bytes of a row in a CTA's shared memory, of which an SM then has four or more, and at most, where eight CTAs have a row: 512 rows of 130000
// logits in 32 bits 115 us, read twice 120; 1024 of 130001 in 16 bits 119 as eight parts, 126 as four.
constexpr long long kPartBytes = 56 * 1024, kMostPartBytes = 72 * 1024;
// Bytes of a row that a warp takes at most; a lane then has 16 packs.  (16384 rows of 2000 logits in 16 bits 31 us, 49 by CTAs; 8192 of 3500
// 30 and 33.)
constexpr long long kWarpBytes = 8192;
template <typename T>
void launch_rows(const ffcvb_cross_entropy_args &a, cudaStream_t stream) {
    constexpr int W = 16 / (int)sizeof(T);
    const uintptr_t apart = reinterpret_cast<uintptr_t>(a.logits) ^ reinterpret_cast<uintptr_t>(a.grad);
    const bool soft = a.target_kind == FFCVB_TARGET_SOFT, both = a.grad && !a.from_stats; // (both passes)
    Deal deal{};
    deal.wide = !a.grad || ((apart & 15) == 0 && (a.logits_stride - a.grad_stride) % W == 0);
    // probabilities lie to 16-byte boundaries as the logits' packs do: strides differ by whole packs, both begin on one
    deal.soft_wide = soft && ((reinterpret_cast<uintptr_t>(a.logits) | reinterpret_cast<uintptr_t>(a.target)) & 15) == 0 &&
                     (a.logits_stride - a.target_stride) % W == 0;
    const long long packs = deal.wide ? a.classes / W : 0; // (at most)
    cudaLaunchConfig_t how{};
    cudaLaunchAttribute with[2] = {};
    how.stream = stream;
    how.attrs = with;
    with[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    with[0].val.programmaticStreamSerializationAllowed = 1;
    how.numAttrs = 1;
    auto run = [&](auto kernel) {
        if (how.dynamicSmemBytes > 40 * 1024) {
            // (the limit is the kernel's, not the call's: another thread's call that needs less must not lower it)
            cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMostPartBytes);
            cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
        }
        cudaLaunchKernelEx(&how, kernel, a, deal);
    };
    if (a.classes * (long long)sizeof(T) <= kWarpBytes) {
        // lanes of a row: one for every two packs, or for every two logits where there are no packs
        const long long pieces = packs ? packs : a.classes;
        const int lanes = pieces <= 4 ? 2 : pieces <= 16 ? 8 : 32;
        deal.part = (int)packs;
        how.gridDim = dim3((unsigned)((a.rows * lanes + 127) / 128));
        how.blockDim = dim3(128);
        how.dynamicSmemBytes = both ? 128 / lanes * packs * 16 : 0;
        auto by_lanes = [&](auto n) {
            constexpr int L = decltype(n)::value;
            if (both)
                run(soft ? rows_kernel<T, true, true, L> : rows_kernel<T, true, false, L>);
            else
                run(soft ? rows_kernel<T, false, true, L> : rows_kernel<T, false, false, L>);
        };
        if (lanes == 2)
            by_lanes(std::integral_constant<int, 2>{});
        else if (lanes == 8)
            by_lanes(std::integral_constant<int, 8>{});
        else
            by_lanes(std::integral_constant<int, 32>{});
        return;
    }
    // CTAs per row: until a part fits, and until there are two CTAs per SM (with few rows) of parts that are worth it
    int ctas = 1;
    while (ctas < 8 && ((both && (packs + ctas - 1) / ctas * 16 > kPartBytes) || (a.rows * ctas <= kSms && packs > 2048 * ctas))) ctas *= 2;
    deal.part = (int)((packs + ctas - 1) / ctas);
    const bool staged = both && deal.part * 16ll <= kMostPartBytes; // (else the second pass reads what the caches still have)
    const int threads = (deal.part / 14 + 31) / 32 * 32; // (14 packs each: 131 us for 8192 x 21841 in bf16, 134 with 16, 136 with 18)
    how.gridDim = dim3((unsigned)(a.rows * ctas));
    how.blockDim = dim3(!deal.wide || threads > 256 ? 256 : threads < 64 ? 64 : threads);
    how.dynamicSmemBytes = staged ? deal.part * 16ll : 0;
    if (ctas > 1) {
        cudaLaunchAttribute &cluster = with[how.numAttrs++];
        cluster.id = cudaLaunchAttributeClusterDimension;
        cluster.val.clusterDim.x = ctas;
        cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
    }
    if (staged)
        run(soft ? rows_kernel<T, true, true, 0> : rows_kernel<T, true, false, 0>);
    else
        run(soft ? rows_kernel<T, false, true, 0> : rows_kernel<T, false, false, 0>);
}

} // namespace

void launch_mean(const float *row_loss, int64_t rows, const float *counted, bool mean, float *loss, cudaStream_t stream) {
    launch_early(mean_kernel, 1, 1024, 0, stream, row_loss, rows, counted, mean, loss);
}
void launch_count(const void *labels, int64_t rows, int64_t stride, int64_t ignore, float *counted, cudaStream_t stream) {
    launch_early(count_kernel, 1, 1024, 0, stream, static_cast<const int64_t *>(labels), rows, stride, ignore, counted);
}

} // namespace ffcvb

using namespace ffcvb;

extern "C" int ffcvb_cross_entropy(const ffcvb_cross_entropy_args *args, void *stream) {
    if (!args) return training_fail(FFCVB_E_ARG, "ffcvb_cross_entropy: no arguments");
    const ffcvb_cross_entropy_args &a = *args;
    // (classes are counted in 32 bits, by steps of up to 4 * 8 * 256 behind the last one)
    if (a.rows < 0 || a.classes < 1 || a.rows > 0x0fffffff || a.classes > 0x7fff0000 || (a.type != FFCVB_TYPE_F32 && a.type != FFCVB_TYPE_F16 && a.type != FFCVB_TYPE_BF16))
        return training_fail(FFCVB_E_ARG, "ffcvb_cross_entropy: bad size or type");
    const bool needs_count = a.has_ignore && a.mean && a.target_kind == FFCVB_TARGET_LABELS;
    if (a.target_kind < FFCVB_TARGET_LABELS || a.target_kind > FFCVB_TARGET_SOFT || !(a.smoothing >= 0.0f && a.smoothing <= 1.0f) ||
        (a.rows > 0 && (!a.logits || !a.target || (a.from_stats ? !a.stats || !a.grad : !a.row_loss))) || (needs_count && !a.counted) ||
        (a.has_ignore && a.target_kind != FFCVB_TARGET_LABELS))
        return training_fail(FFCVB_E_ARG, "ffcvb_cross_entropy: bad argument");
    if ((reinterpret_cast<uintptr_t>(a.stats) & 7) != 0) return training_fail(FFCVB_E_ARG, "ffcvb_cross_entropy: stats begin on 8 bytes");
    OnDevice here(a.device);
    if (!here.ok()) return training_fail(FFCVB_E_NODEVICE, "ffcvb_cross_entropy: no device %d", a.device);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (needs_count) launch_count(a.target, a.rows, a.target_stride, a.ignore_index, a.counted, st);
    if (a.rows > 0) with_type(a.type, [&](auto zero) { launch_rows<decltype(zero)>(a, st); });
    if (a.loss && !a.from_stats) launch_mean(a.row_loss, a.rows, needs_count ? a.counted : nullptr, a.mean, a.loss, st);
    return launched("ffcvb_cross_entropy");
}
