// Cross entropy against labels, mixed labels or probabilities, with its gradient (sm_100a).
//
// With T the target's probabilities, S their sum and lse = log sum exp x, a row's loss is S * lse - sum T x and
// its gradient S * exp(x - lse) - T.  One CTA takes a row: a pass over the logits keeps each thread's maximum and
// the sum of exponentials relative to it (in 32 bits), which are joined over the CTA; a second pass, whose reads come from
// L2, writes the gradient.
#include "training.h"

namespace ffcvb {

namespace {

// (Differences are taken before the factor: a row masked with the type's lowest value has no product with it.)
__device__ __forceinline__ float exp_of(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * 1.4426950408889634f));
    return y;
}

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

template <int WARPS>
__device__ __forceinline__ float cta_sum(float v, float *s) {
    v = warp_sum(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    return warp_sum((threadIdx.x & 31) < WARPS ? s[threadIdx.x & 31] : 0.0f);
}
template <int WARPS>
__device__ __forceinline__ float cta_max(float v, float *s) {
    v = warp_max(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    return warp_max((threadIdx.x & 31) < WARPS ? s[threadIdx.x & 31] : -INFINITY);
}

__device__ __forceinline__ float probability(const ffcvb_cross_entropy_args &a, long long at) {
    switch (a.target_type) {
    case FFCVB_TYPE_F16: return to_float(static_cast<const __half *>(a.target)[at]);
    case FFCVB_TYPE_BF16: return to_float(static_cast<const __nv_bfloat16 *>(a.target)[at]);
    }
    return static_cast<const float *>(a.target)[at];
}

// One row per CTA.  WIDE: 16 bytes at a time from the 16-byte boundary at or before the row on (what lies before
// the row there is left out); logits and gradient then lie alike to these boundaries.
template <typename T, int THREADS, bool WIDE, bool SOFT>
__global__ void __launch_bounds__(THREADS)
rows_kernel(const __grid_constant__ ffcvb_cross_entropy_args a) {
    constexpr int N = WIDE ? kWide<T> : 1;
    constexpr int WARPS = THREADS / 32;
    __shared__ float s_part[32];
    const long long row = blockIdx.x;
    const long long classes = a.classes;
    const T *x = static_cast<const T *>(a.logits) + row * a.logits_stride;
    T *g = a.grad ? static_cast<T *>(a.grad) + row * a.grad_stride : nullptr;
    const Picks p = picks_of(a, row);
    if (p.ignored || p.bad) {
        const float v = p.ignored ? 0.0f : NAN;
        if (g)
            for (long long c = threadIdx.x; c < classes; c += THREADS) g[c] = from_float<T>(v);
        if (threadIdx.x == 0 && !a.from_stats) {
            a.row_loss[row] = v;
            if (a.stats) reinterpret_cast<float2 *>(a.stats)[row] = make_float2(v, v);
        }
        return;
    }
    const int lead = WIDE ? (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T)) : 0;
    const long long packs = (lead + classes + N - 1) / N;
    const T *x0 = x - lead;
    const long long soft_row = row * a.target_stride;
    const float sure = 1.0f - a.smoothing;

    float row_top, over, total = p.total; // (over: 1 / sum of exp(x - row_top), 0 where there is nothing)
    if (!a.from_stats) {
        float top = -INFINITY, sum = 0.0f, dot = 0.0f, mass = 0.0f;
        for (long long k = threadIdx.x; k < packs; k += THREADS) {
            Pack<T, N> pack;
            pack.load(x0 + k * N);
            float v[N];
            pack.get(v);
            float most = top;
#pragma unroll
            for (int j = 0; j < N; j++) {
                const long long c = k * N + j - lead;
                if (c < 0 || c >= classes) {
                    v[j] = -INFINITY;
                    continue;
                }
                most = fmaxf(most, v[j]);
                if (SOFT || p.flat > 0.0f) {
                    const float t = SOFT ? sure * probability(a, soft_row + c) + p.flat : p.flat;
                    if (SOFT) mass += t;
                    if (t > 0.0f) dot += t * v[j];
                }
            }
            if (top != -INFINITY) sum *= exp_of(top - most);
            const float base = most == -INFINITY ? 0.0f : most;
            float part = exp_of(v[0] - base);
#pragma unroll
            for (int j = 1; j < N; j++) part += exp_of(v[j] - base);
            sum += part;
            top = most;
        }
        row_top = cta_max<WARPS>(top, s_part);
        if (top != -INFINITY) sum *= exp_of(top - row_top);
        if (row_top == -INFINITY) row_top = 0.0f;
        sum = cta_sum<WARPS>(sum, s_part);
        over = sum == 0.0f ? 0.0f : 1.0f / sum;
        if (SOFT || p.flat > 0.0f) dot = cta_sum<WARPS>(dot, s_part);
        if (SOFT) total = cta_sum<WARPS>(mass, s_part);
        if (threadIdx.x == 0) {
#pragma unroll
            for (int k = 0; k < 2; k++)
                if (p.weight[k] != 0.0f) dot += p.weight[k] * to_float(x[p.label[k]]);
            a.row_loss[row] = sum == 0.0f ? 0.0f : total * (row_top + logf(sum)) - dot;
            if (a.stats) reinterpret_cast<float2 *>(a.stats)[row] = make_float2(row_top, over);
        }
    } else {
        const float2 stats = reinterpret_cast<const float2 *>(a.stats)[row];
        row_top = stats.x;
        over = stats.y;
        if (SOFT) {
            float mass = 0.0f;
            for (long long c = threadIdx.x; c < classes; c += THREADS) mass += sure * probability(a, soft_row + c) + p.flat;
            total = cta_sum<WARPS>(mass, s_part);
        }
    }
    if (!g) return;
    float k_row = a.scale;
    if (a.upstream) k_row *= a.upstream[a.upstream_per_row ? row : 0];
    if (a.mean) k_row /= a.has_ignore ? fmaxf(a.counted[0], 1.0f) : (float)a.rows;
    if (over == 0.0f) k_row = 0.0f;
    const float factor = k_row * total * over;
    T *g0 = g - lead;
    for (long long k = threadIdx.x; k < packs; k += THREADS) {
        Pack<T, N> pack;
        pack.load(x0 + k * N);
        float v[N];
        pack.get(v);
#pragma unroll
        for (int j = 0; j < N; j++) {
            const long long c = k * N + j - lead;
            float t = p.flat;
            if (SOFT) t += c >= 0 && c < classes ? sure * probability(a, soft_row + c) : 0.0f;
            if (c == p.label[0]) t += p.weight[0];
            if (c == p.label[1]) t += p.weight[1];
            v[j] = factor * exp_of(v[j] - row_top) - k_row * t;
        }
        pack.set(v);
        if (!WIDE || (k * N >= lead && k * N + N - lead <= classes)) {
            pack.store(g0 + k * N);
        } else {
#pragma unroll
            for (int j = 0; j < N; j++) {
                const long long c = k * N + j - lead;
                if (c >= 0 && c < classes) g[c] = from_float<T>(v[j]);
            }
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

template <typename T>
void launch_rows(const ffcvb_cross_entropy_args &a, cudaStream_t stream) {
    const uintptr_t apart = reinterpret_cast<uintptr_t>(a.logits) ^ reinterpret_cast<uintptr_t>(a.grad);
    const bool wide = !a.grad || ((apart & 15) == 0 && (a.logits_stride - a.grad_stride) * (long long)sizeof(T) % 16 == 0);
    const bool soft = a.target_kind == FFCVB_TARGET_SOFT;
    auto run = [&](auto kernel) { kernel<<<(unsigned)a.rows, 256, 0, stream>>>(a); };
    if (wide)
        run(soft ? rows_kernel<T, 256, true, true> : rows_kernel<T, 256, true, false>);
    else
        run(soft ? rows_kernel<T, 256, false, true> : rows_kernel<T, 256, false, false>);
}

} // namespace

} // namespace ffcvb

using namespace ffcvb;

extern "C" int ffcvb_cross_entropy(const ffcvb_cross_entropy_args *args, void *stream) {
    if (!args) return training_fail(FFCVB_E_ARG, "ffcvb_cross_entropy: no arguments");
    const ffcvb_cross_entropy_args &a = *args;
    if (a.rows < 0 || a.classes < 1 || a.rows > 0x7fffffff || (a.type != FFCVB_TYPE_F32 && a.type != FFCVB_TYPE_F16 && a.type != FFCVB_TYPE_BF16))
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
