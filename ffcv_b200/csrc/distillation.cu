// Distillation from a teacher's largest logits, with its gradient (sm_100a).
//
// A row's teacher gives `kept` classes c_k with logits t_k; q = softmax(t / tau) over them.  With p = softmax(x / tau) over all classes the soft loss is
// tau^2 sum q (log q - log p_c), its gradient tau (Q p - q) with Q = 1, or 0 where no entry is left; the hard loss is the cross entropy of the same
// logits (see cross_entropy.cu), and both are added with weights 1 - h and h.
//
// A warp takes a row of up to 8 KB and 32 entries, a CTA one of up to 56 KB, a cluster a longer one.  Every thread copies its part of the row into shared
// memory, in places of its own; a pass over it keeps the largest logit so far and the sums of exponentials relative to it at both temperatures, which
// are joined over the row's threads together with the teacher's; a second pass makes the part of the gradient that all classes have; then the
// classes with entries, or labels, are written once more, each by one thread, with the shares of all entries of that class, in their order: the same
// class may come twice.  So the row crosses HBM once each way.
//
// What bounds it: exponentials and the instructions around them, and that a row's passes wait for one another.  A logit has two exponentials, one in each pass; four with the hard loss, but
// where the temperature is 1, 2 or 4, whose one exponential gives the other.  8192 x 21841 bf16 logits with 64 entries take 158 to 164 us, 110 at the rate of a copy; the unit for exponentials
// is busy for 67 % of it and 65 % of the turns to issue are used, by five CTAs on an SM, whose warps wait for one another's results and at barriers most.  1531 x 50021 fp16 logits with 200
// entries and labels at 3.5 take 118 to 121 us, 47 at the rate of a copy (80 % of the unit's time with 8192 x 21841).  512 x 10 take 8 us: two launches.
#include "losses.h"

#include <algorithm>
#include <type_traits>

namespace ffcvb {

namespace {

constexpr int kMostKept = FFCVB_DISTILLATION_MOST;

// Of a part of a row: the largest logit, at least kLowest; sums of exponentials relative to it, at the temperature and (HARD) at 1; with smoothing what its classes have of the
// target, and the sum of that times the logits relative to the largest (of differences themselves to logits of the type's lowest value, which mask classes, it would not be finite).
struct Sums {
    float top, soft, hard, away, mass;
    static __device__ __forceinline__ float shift(float mass, float from, float to) { return mass * fmaxf(from - to, kLowest); }
    __device__ __forceinline__ void to(float most, float rate) {
        soft *= exp2_of((top - most) * rate);
        hard *= exp_of(top - most);
        away += shift(mass, top, most);
        top = most;
    }
    __device__ __forceinline__ void join(Sums o, float rate) {
        const float most = fmaxf(top, o.top);
        to(most, rate);
        o.to(most, rate);
        soft += o.soft;
        hard += o.hard;
        away += o.away;
        mass += o.mass;
    }
    // joins those of groups of LANES lanes
    template <int LANES, int HARD> __device__ __forceinline__ void join_lanes(float rate, bool spread) {
        float most = top;
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        soft *= exp2_of((top - most) * rate);
        if (HARD) hard *= exp_of(top - most);
        if (spread) away += shift(mass, top, most);
        top = most;
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) {
            soft += __shfl_xor_sync(0xffffffffu, soft, o);
            if (HARD) hard += __shfl_xor_sync(0xffffffffu, hard, o);
        }
        if (!spread) return;
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) {
            away += __shfl_xor_sync(0xffffffffu, away, o);
            mass += __shfl_xor_sync(0xffffffffu, mass, o);
        }
    }
};

// The same of the teacher's logits, at the temperature.  (Differences are divided by it, not logits: one below 1 would leave the type's lowest value infinite.)
struct Given {
    float top, sum;
    __device__ __forceinline__ void add(float t, float rate) {
        const float most = fmaxf(top, t);
        sum = sum * exp2_of((top - most) * rate) + exp2_of((t - most) * rate);
        top = most;
    }
    template <int LANES> __device__ __forceinline__ void join_lanes(float rate) {
        float most = top;
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        sum *= exp2_of((top - most) * rate);
        top = most;
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
};

__device__ __forceinline__ long long class_of(const ffcvb_distillation_args &a, long long row, int k) {
    const long long at = row * a.classes_stride + k;
    return a.classes_wide ? static_cast<const int64_t *>(a.teacher_classes)[at] : static_cast<const int32_t *>(a.teacher_classes)[at];
}
__device__ __forceinline__ float logit_of(const ffcvb_distillation_args &a, long long row, int k) {
    const long long at = row * a.teacher_stride + k;
    return a.teacher_type == FFCVB_TYPE_F32   ? static_cast<const float *>(a.teacher)[at]
           : a.teacher_type == FFCVB_TYPE_F16 ? to_float(static_cast<const __half *>(a.teacher)[at])
                                              : to_float(static_cast<const __nv_bfloat16 *>(a.teacher)[at]);
}

// How rows are dealt out: whether logits and gradient lie alike to 16-byte boundaries; packs of a CTA's part of a row.
struct Deal {
    int wide, part;
};

// The loss against labels: none; with exponentials of its own; or with those at the temperature, to the power of 1, 2 or 4, which the temperature then is (two instead of
// four exponentials for a logit).
enum { kNoHard, kOwn, kFirst, kSecond, kFourth };
template <int HARD> __device__ __forceinline__ float hard_exp(float d, float soft) {
    return HARD == kFirst ? soft : HARD == kSecond ? soft * soft : HARD == kFourth ? (soft * soft) * (soft * soft) : exp_of(d);
}
template <int HARD> __device__ __forceinline__ Two hard_exp(Two d, Two soft) {
    if constexpr (HARD == kFirst) return soft;
    if constexpr (HARD == kSecond) return mul_rn(soft, soft);
    if constexpr (HARD == kFourth) return mul_rn(mul_rn(soft, soft), mul_rn(soft, soft));
    const Two h = mul_rn(d, Two(kLog2e, kLog2e));
    return Two(exp2_of(h.lo()), exp2_of(h.hi()));
}

// WARP: a row per warp, one entry per lane, in CTAs of four; else a row per CTA or cluster.  STAGED: packs go through shared memory; else they are read
// where they are needed.  HARD: with the loss against labels.
template <typename T, bool STAGED, bool WARP, int HARD>
__global__ void __launch_bounds__(WARP ? 128 : 256)
distill_kernel(const __grid_constant__ ffcvb_distillation_args a, const Deal deal) {
    constexpr int N = kWide<T>, BATCH = STAGED ? 1 : 4; // packs that a thread has on their way
    __shared__ float s_part[8][8], s_there[8][8];       // of the CTA's warps, of the cluster's CTAs
    __shared__ int s_bad;
    extern __shared__ uint4 s_row[];
    wait_for_previous();
    let_next_begin();
    uint32_t rank = 0, ranks = 1;
    if (!WARP) {
        asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
        asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
        if (ranks > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); // (this one has begun)
    }
    const int thread = WARP ? threadIdx.x & 31 : threadIdx.x, threads = WARP ? 32 : blockDim.x, lane = threadIdx.x & 31;
    const long long row = WARP ? blockIdx.x * 4ll + threadIdx.x / 32 : blockIdx.x / ranks;
    if (WARP && row >= a.rows) return;
    const int classes = (int)a.classes, kept = (int)a.kept;
    const T *x = static_cast<const T *>(a.logits) + row * a.logits_stride;
    T *g = a.grad ? static_cast<T *>(a.grad) + row * a.grad_stride : nullptr;
    // logits before the packs, packs of the row and of this CTA's part, logits besides packs
    const int lead = (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / (int)sizeof(T);
    const int before = deal.wide && lead < classes ? lead : classes;
    const int packs = (classes - before) / N, singles = classes - packs * N;
    const int first = (int)rank * deal.part, count = max(0, min(packs - first, deal.part));
    const T *x0 = x + before + (long long)first * N;
    // before the row's packs: entries' classes, teacher's logits, own logits; of each thread a list of those entries whose classes it writes
    int *s_class = reinterpret_cast<int *>(s_row), *s_next = s_class + 3 * kept, *s_first = s_next + kept;
    float *s_given = reinterpret_cast<float *>(s_class + kept), *s_logit = s_given + kept;
    const int head = WARP ? 0 : (4 * kept + threads + 3) / 4;
    // (a CTA's threads keep their first pack in registers: so much less shared memory, five CTAs of 21841 logits on an SM and not four)
    constexpr bool OWN = STAGED && !WARP;
    const uint32_t mine = (uint32_t)__cvta_generic_to_shared(s_row + head + (WARP ? threadIdx.x / 32 * deal.part : 0) + thread) - (OWN ? threads * 16 : 0);
    Pack<T, N> own;
    if (STAGED) {
        uint32_t to = mine;
        for (int k = thread; k < count; k += threads, to += threads * 16) {
            if (OWN && k == thread)
                own.load(x0 + (long long)k * N);
            else
                copy16(to, x0 + (long long)k * N);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    auto single = [&](int k) { return k < before ? k : k + packs * N; }; // class of the k-th besides packs
    Picks p{{-1, -1}, {0.0f, 0.0f}, 0.0f, 0.0f, false, false};
    if (a.target) {
        p = picks_of(a, row);
        if (!HARD) p.bad = false;
    }
    // The row's entries.  A class above the last one makes the row bad, one below 0 is no entry.
    const float tau = a.temperature, rate = kLog2e / tau;
    Given given{kLowest, 0.0f};
    int my_class = -1; // (WARP)
    float my_logit = 0.0f, my_x = 0.0f;
    bool bad = p.bad;
    if (WARP) {
        if (lane < kept) {
            const long long c = class_of(a, row, lane);
            bad |= c >= classes;
            my_class = c < 0 || c >= classes ? -1 : (int)c;
            if (my_class >= 0) {
                my_x = to_float(x[my_class]);
                given.add(my_logit = logit_of(a, row, lane), rate);
            }
        }
        bad = __any_sync(0xffffffffu, bad);
        given.join_lanes<32>(rate);
    } else {
        if (thread == 0) s_bad = 0;
        s_first[thread] = -1;
        __syncthreads();
    }
    // The thread that writes a class, or -1: one of another CTA.
    auto writer = [&](int c) {
        const int in = c - before;
        if (in >= 0 && in < packs * N) {
            const int mine = in / N - first;
            return mine < 0 || mine >= count ? -1 : mine % threads;
        }
        const int k = in < 0 ? c : c - packs * N;
        return k / threads % (int)ranks == (int)rank ? k % threads : -1;
    };
    // (WARP not:) A thread's first entry is loaded ahead, its class at once, its logit here once the row is, and taken behind the first pass.
    const long long ahead = !WARP && thread < kept ? class_of(a, row, thread) : -1;
    float ahead_logit = !WARP && thread < kept ? logit_of(a, row, thread) : 0.0f, ahead_x = 0.0f;
    auto take_entry = [&](int k, long long c, float t, float v) {
        bad |= c >= classes;
        const int here = c < 0 || c >= classes || t == -INFINITY ? -1 : (int)c; // (rows that are filled up with one class have no long lists)
        s_class[k] = here;
        if (here < 0) return;
        s_given[k] = t;
        s_logit[k] = v;
        given.add(t, rate);
        const int by = writer(here);
        if (by >= 0) s_next[k] = atomicExch(s_first + by, k);
    };
    auto load_ahead = [&] {
        if (!WARP && ahead >= 0 && ahead < classes) ahead_x = to_float(x[ahead]);
    };
    auto take_entries = [&] {
        if (WARP) return;
        if (thread < kept) take_entry(thread, ahead, ahead_logit, ahead_x);
        for (int k = thread + threads; k < kept; k += threads) {
            const long long c = class_of(a, row, k);
            take_entry(k, c, logit_of(a, row, k), c >= 0 && c < classes ? to_float(x[c]) : 0.0f);
        }
        if (bad) s_bad = 1;
        given.join_lanes<32>(rate);
    };
    if (p.ignored) { // (all of a row's threads alike)
        const T zero = from_float<T>(0.0f);
        if (g)
            for (int c = (int)rank * threads + thread; c < classes; c += (int)ranks * threads) g[c] = zero;
        if (thread == 0 && rank == 0 && !a.from_stats) {
            a.row_loss[row] = 0.0f;
            if (a.stats) reinterpret_cast<float4 *>(a.stats)[row] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
        if (STAGED) asm volatile("cp.async.wait_group 0;" ::: "memory");
        if (ranks > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
        return;
    }
    // Calls f(values, class of the first) for this thread's packs: as many turns as all threads have, BATCH at a time, then what is left.
    const int turns = count / threads;
    auto each_pack = [&](auto &&f) {
        uint32_t at = mine;
        const T *from = x0 + (long long)thread * N;
        int c = before + (first + thread) * N;
        const int step = threads * N;
        int k = 0;
        auto load = [&](Pack<T, N> &pack, int i) {
            if (OWN && k + i == 0) {
                pack = own;
            } else if constexpr (STAGED) {
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
    const bool spread = HARD && p.flat > 0.0f;
    Sums sums{kLowest, 0.0f, 0.0f, 0.0f, 0.0f};
    if (!a.from_stats) {
        auto take = [&](auto &v, int) {
            constexpr int M = sizeof(v) / 4;
            float most = fmaxf(sums.top, v[0]);
#pragma unroll
            for (int j = 1; j < M; j++) most = fmaxf(most, v[j]);
            const float less = sums.top - most;
            sums.soft *= exp2_of(less * rate);
            if (HARD) sums.hard *= exp_of(less);
            if (spread) sums.away += Sums::shift(sums.mass, sums.top, most);
            sums.top = most;
            if constexpr (M == 1) {
                const float d = v[0] - most, e = exp2_of(d * rate);
                sums.soft += e;
                if (HARD) sums.hard += hard_exp<HARD>(d, e);
                if (spread) sums.away += p.flat * d;
            } else {
                const Two minus(-most, -most), rates(rate, rate), flat(p.flat, p.flat);
                Two soft(0.0f, 0.0f), hard(0.0f, 0.0f), away(0.0f, 0.0f);
#pragma unroll
                for (int j = 0; j < M; j += 2) {
                    const Two d = add_rn(Two(v[j], v[j + 1]), minus), s = mul_rn(d, rates);
                    const Two e(exp2_of(s.lo()), exp2_of(s.hi()));
                    soft = add_rn(soft, e);
                    if (HARD) hard = add_rn(hard, hard_exp<HARD>(d, e));
                    if (spread) away = fma_rn(d, flat, away);
                }
                sums.soft += soft.lo() + soft.hi();
                if (HARD) sums.hard += hard.lo() + hard.hi();
                if (spread) sums.away += away.lo() + away.hi();
            }
            if (spread) sums.mass += M * p.flat;
        };
        each_single([&](int c) {
            const float v[1] = {to_float(x[c])};
            take(v, c);
        });
        if (STAGED) asm volatile("cp.async.wait_group 0;" ::: "memory");
        load_ahead();
        each_pack(take);
        take_entries();
        sums.join_lanes<32, HARD>(rate, spread);
    } else {
        load_ahead();
        take_entries();
    }
    if (!WARP) {
        const int warps = blockDim.x >> 5;
        if (lane == 0) {
            float *to = s_part[threadIdx.x >> 5];
            to[0] = sums.top, to[1] = sums.soft, to[2] = sums.hard, to[3] = sums.away, to[4] = sums.mass, to[5] = given.top, to[6] = given.sum;
        }
        __syncthreads();
        const float *from = s_part[lane & 7];
        const bool there = (lane & 7) < warps; // (at most eight)
        sums = there ? Sums{from[0], from[1], from[2], from[3], from[4]} : Sums{kLowest, 0.0f, 0.0f, 0.0f, 0.0f};
        given = there ? Given{from[5], from[6]} : Given{kLowest, 0.0f};
        sums.join_lanes<8, HARD>(rate, spread);
        given.join_lanes<8>(rate);
        bad = s_bad != 0;
        if (ranks > 1) {
            asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); // all have begun
            if (threadIdx.x < ranks) {
                uint32_t to;
                asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"((uint32_t)__cvta_generic_to_shared(s_there[rank])), "r"(threadIdx.x));
                const float v[5] = {sums.top, sums.soft, sums.hard, sums.away, sums.mass};
#pragma unroll
                for (int i = 0; i < 5; i++) asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 4 * i), "f"(v[i]) : "memory");
            }
            asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
            sums = Sums{s_there[0][0], s_there[0][1], s_there[0][2], s_there[0][3], s_there[0][4]};
            for (uint32_t k = 1; k < ranks; k++) sums.join(Sums{s_there[k][0], s_there[k][1], s_there[k][2], s_there[k][3], s_there[k][4]}, rate);
        }
    }
    float over_soft, over_hard; // 1 / sums, 0 where there is nothing
    if (a.from_stats) {
        const float4 stats = reinterpret_cast<const float4 *>(a.stats)[row];
        sums.top = stats.x;
        over_soft = stats.y;
        over_hard = stats.z;
    } else {
        over_soft = sums.soft == 0.0f ? 0.0f : 1.0f / sums.soft;
        over_hard = !HARD || sums.hard == 0.0f ? 0.0f : 1.0f / sums.hard;
        if (bad) over_soft = over_hard = NAN;
        if (thread == 0 && rank == 0 && a.stats) reinterpret_cast<float4 *>(a.stats)[row] = make_float4(sums.top, over_soft, over_hard, 0.0f);
    }
    const float top = sums.top, hard = HARD ? a.hard : 0.0f, soft = 1.0f - hard;
    const float all = given.sum == 0.0f ? 0.0f : 1.0f, over_given = given.sum == 0.0f ? 0.0f : 1.0f / given.sum;
    float k_row = a.scale;
    if (a.upstream) k_row *= a.upstream[a.upstream_per_row ? row : 0];
    if (a.mean) k_row /= a.counted ? fmaxf(*a.counted, 1.0f) : (float)a.rows;
    const bool blank = over_soft == 0.0f; // (no logit but -inf)
    if (blank) k_row = 0.0f;
    const float k_soft = k_row * soft * tau, k_hard = k_row * hard;
    const float times_soft = bad ? NAN : k_soft * all * over_soft, times_hard = k_hard * p.total * over_hard, flat = k_hard * p.flat;
    // what a class has of the gradient besides entries and labels
    auto common = [&](float v) {
        const float d = v - top, e = exp2_of(d * rate);
        float out = times_soft * e - flat;
        if (HARD) out += times_hard * hard_exp<HARD>(d, e);
        return out;
    };
    auto share_of = [&](float t) { return exp2_of((t - given.top) * rate) * over_given; };
    if (thread < 32 && rank == 0 && !a.from_stats) { // a warp has the loss
        // the soft one is tau^2 sum q (log q - log p); log q has the teacher's sum, log p the student's, both once for all shares
        float loss = 0.0f;
        auto add = [&](float t, float v) {
            const float q = share_of(t);
            if (q != 0.0f) loss += q * ((t - given.top) - (v - top));
        };
        if (WARP) {
            if (my_class >= 0) add(my_logit, my_x);
        } else {
            for (int k = lane; k < kept; k += 32)
                if (s_class[k] >= 0) add(s_given[k], s_logit[k]);
        }
        loss = warp_sum(loss);
        if (lane == 0) {
            float out = soft == 0.0f || all == 0.0f ? 0.0f : soft * tau * (loss + tau * (logf(sums.soft) - logf(given.sum)));
            if (HARD) {
                float dot = spread ? sums.away : 0.0f;
#pragma unroll
                for (int k = 0; k < 2; k++)
                    if (p.weight[k] != 0.0f && !bad) dot += p.weight[k] * (to_float(x[p.label[k]]) - top);
                out += hard * (p.total * logf(sums.hard) - dot);
            }
            a.row_loss[row] = bad ? NAN : blank ? 0.0f : out;
        }
    }
    if (!g) return;
    {
        each_single([&](int c) { g[c] = from_float<T>(common(to_float(x[c]))); });
        const Two minus(-top, -top), rates(rate, rate), less(-flat, -flat), soft2(times_soft, times_soft), hard2(times_hard, times_hard);
        each_pack([&](float(&v)[N], int c) {
#pragma unroll
            for (int j = 0; j < N; j += 2) {
                const Two d = add_rn(Two(v[j], v[j + 1]), minus), s = mul_rn(d, rates);
                const Two e(exp2_of(s.lo()), exp2_of(s.hi()));
                Two out = fma_rn(e, soft2, less);
                if (HARD) out = fma_rn(hard_exp<HARD>(d, e), hard2, out);
                v[j] = out.lo();
                v[j + 1] = out.hi();
            }
            Pack<T, N> pack;
            pack.set(v);
            pack.store(g + c);
        });
    }
    if (bad) return;
    // Classes with entries or labels once more, by the thread that has written them (or the warp), with the shares of all entries of a class in their order.
    auto again = [&](int c, float logit, float share) {
        float v = common(logit) - k_soft * share;
        if (HARD) {
#pragma unroll
            for (int k = 0; k < 2; k++)
                if (c == (int)p.label[k]) v -= k_hard * p.weight[k];
        }
        g[c] = from_float<T>(v);
    };
    bool alone[2]; // labels without an entry, which this thread writes
    if (WARP) {
        __syncwarp();
        const float mine_share = my_class >= 0 ? share_of(my_logit) : 0.0f;
        const uint32_t same = __match_any_sync(0xffffffffu, my_class);
        float share = 0.0f;
        for (int k = 0; k < kept; k++) { // (all lanes take part)
            const float s = __shfl_sync(0xffffffffu, mine_share, k);
            if (same >> k & 1) share += s;
        }
        if (my_class >= 0 && lane == __ffs(same) - 1) again(my_class, my_x, share);
#pragma unroll
        for (int k = 0; k < 2; k++) alone[k] = HARD && !__any_sync(0xffffffffu, my_class >= 0 && my_class == (int)p.label[k]) && thread == k;
    } else {
#pragma unroll
        for (int k = 0; k < 2; k++) alone[k] = HARD && p.label[k] >= 0 && writer((int)p.label[k]) == thread;
        for (int k = s_first[thread]; k >= 0; k = s_next[k]) {
            const int c = s_class[k];
#pragma unroll
            for (int l = 0; l < 2; l++) alone[l] = alone[l] && c != (int)p.label[l];
            bool earlier = false, later = false; // entries of the same class: they are in the same list
            for (int j = s_first[thread]; j >= 0 && !earlier; j = s_next[j])
                if (j != k && s_class[j] == c) (j < k ? earlier : later) = true;
            if (earlier) continue;
            float share = share_of(s_given[k]);
            if (later)
                for (int j = k + 1; j < kept; j++)
                    if (s_class[j] == c) share += share_of(s_given[j]);
            again(c, s_logit[k], share);
        }
    }
    if (HARD) {
#pragma unroll
        for (int k = 0; k < 2; k++)
            if (alone[k] && p.label[k] >= 0 && !(k == 1 && p.label[0] == p.label[1])) again((int)p.label[k], to_float(x[p.label[k]]), 0.0f);
    }
}

// As for the cross entropy's rows: bytes of a row in a CTA's shared memory (8192 x 21841 in 16 bits 156 us, 181 with 40 KB, 157 with 100; 1531 x 50021 124, 132 and
// 124; with 56, 40 and 72 KB 3413 x 24000 87, 89 and 87, 2730 x 30000 86, 86 and 93, 1637 x 50021 91, 88 and 91, 1170 x 70000 87, 87 and 92, 409 x 200000 89 each, in
// 32 bits 4818 x 17000 139, 140 and 142, 3750 x 21841 142, 150 and 142), at most where eight CTAs have a row, and in a warp's (16384 x 2000 in 16 bits 54 us, 88 by CTAs; 8192 x 3500 35 and 45; 16384 x 300 in 32 bits 27 and 73).
constexpr long long kPartBytes = 56 * 1024, kMostPartBytes = 72 * 1024, kWarpBytes = 8192;

template <typename T, int HARD> void launch_rows(const ffcvb_distillation_args &a, cudaStream_t stream) {
    constexpr int W = 16 / (int)sizeof(T);
    const uintptr_t apart = reinterpret_cast<uintptr_t>(a.logits) ^ reinterpret_cast<uintptr_t>(a.grad);
    const bool both = a.grad && !a.from_stats; // (both passes)
    Deal deal{};
    deal.wide = !a.grad || ((apart & 15) == 0 && (a.logits_stride - a.grad_stride) % W == 0);
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
            cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMostPartBytes + 32 * 1024);
            cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
        }
        cudaLaunchKernelEx(&how, kernel, a, deal);
    };
    if (a.classes * (long long)sizeof(T) <= kWarpBytes && a.kept <= 32) {
        deal.part = (int)packs;
        how.gridDim = dim3((unsigned)((a.rows + 3) / 4));
        how.blockDim = dim3(128);
        how.dynamicSmemBytes = both ? 4 * packs * 16 : 0;
        if (both)
            run(distill_kernel<T, true, true, HARD>);
        else
            run(distill_kernel<T, false, true, HARD>);
        return;
    }
    // CTAs per row: until a part fits, and until there is one for every SM (with few rows) of parts that are worth it (the loss alone of 8 x 200000 10.4 us, 18.5 by a
    // CTA for each row; 8 x 24000 10.4 by two, 8.4 by one; 64 x 50000 10.4 either way)
    int ctas = 1;
    while (ctas < 8 && ((both && (packs + ctas - 1) / ctas * 16 > kPartBytes) || (a.rows * ctas <= kSms && packs > 4096 * ctas))) ctas *= 2;
    deal.part = (int)((packs + ctas - 1) / ctas);
    const bool staged = both && deal.part * 16ll <= kMostPartBytes; // (else the second pass reads what the caches still have)
    const int threads = (deal.part / 14 + 31) / 32 * 32; // (20000 x 6000 125 us, 207 by 256 threads each; 4096 x 8000 66 and 88; with 28 packs each within two in a hundred)
    how.gridDim = dim3((unsigned)(a.rows * ctas));
    how.blockDim = dim3(!deal.wide || threads > 256 ? 256 : threads < 64 ? 64 : threads);
    how.dynamicSmemBytes = (4 * a.kept + how.blockDim.x + 3) / 4 * 16 + (staged ? std::max(0, deal.part - (int)how.blockDim.x) * 16ll : 0);
    if (ctas > 1) {
        cudaLaunchAttribute &cluster = with[how.numAttrs++];
        cluster.id = cudaLaunchAttributeClusterDimension;
        cluster.val.clusterDim.x = ctas;
        cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
    }
    if (staged)
        run(distill_kernel<T, true, false, HARD>);
    else
        run(distill_kernel<T, false, false, HARD>);
}

const char *wrong(const ffcvb_distillation_args &a) {
    auto known = [](int type) { return type == FFCVB_TYPE_F32 || type == FFCVB_TYPE_F16 || type == FFCVB_TYPE_BF16; };
    // (classes are counted in 32 bits, by steps of up to 4 * 8 * 256 behind the last one)
    if (a.rows < 0 || a.classes < 1 || a.rows > 0x0fffffff || a.classes > 0x7fff0000 || a.kept < 1 || a.kept > kMostKept || !known(a.type) || !known(a.teacher_type))
        return "bad size or type";
    if (!(a.temperature >= 1e-30f && a.temperature <= 1e30f) || !(a.hard >= 0.0f && a.hard <= 1.0f) || !(a.smoothing >= 0.0f && a.smoothing <= 1.0f)) return "bad number";
    if (a.target_kind != FFCVB_TARGET_LABELS && a.target_kind != FFCVB_TARGET_MIXED) return "bad target";
    if (a.has_ignore && (!a.target || a.target_kind != FFCVB_TARGET_LABELS)) return "a label to ignore goes with labels";
    if (a.rows > 0 && (!a.logits || !a.teacher || !a.teacher_classes || (a.hard > 0.0f && !a.target) || (a.from_stats ? !a.stats || !a.grad : !a.row_loss)))
        return "an address is missing";
    if (a.has_ignore && a.mean && !a.counted) return "no room for the count";
    if ((reinterpret_cast<uintptr_t>(a.stats) & 15) != 0) return "stats begin on 16 bytes";
    return nullptr;
}

} // namespace

} // namespace ffcvb

using namespace ffcvb;

extern "C" int ffcvb_distillation(const ffcvb_distillation_args *args, void *stream) {
    if (!args) return training_fail(FFCVB_E_ARG, "ffcvb_distillation: no arguments");
    ffcvb_distillation_args a = *args;
    if (const char *what = wrong(a)) return training_fail(FFCVB_E_ARG, "ffcvb_distillation: %s", what);
    OnDevice here(a.device);
    if (!here.ok()) return training_fail(FFCVB_E_NODEVICE, "ffcvb_distillation: no device %d", a.device);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (!(a.has_ignore && a.mean)) a.counted = nullptr;
    if (a.counted) launch_count(a.target, a.rows, a.target_stride, a.ignore_index, a.counted, st);
    if (a.rows > 0)
        with_type(a.type, [&](auto zero) {
            using T = decltype(zero);
            if (!(a.hard > 0.0f))
                launch_rows<T, kNoHard>(a, st);
            else if (a.temperature == 1.0f)
                launch_rows<T, kFirst>(a, st);
            else if (a.temperature == 2.0f)
                launch_rows<T, kSecond>(a, st);
            else if (a.temperature == 4.0f)
                launch_rows<T, kFourth>(a, st);
            else
                launch_rows<T, kOwn>(a, st);
        });
    if (a.loss && !a.from_stats) launch_mean(a.row_loss, a.rows, a.counted, a.mean, a.loss, st);
    return launched("ffcvb_distillation");
}
