// One AdamW step over many tensors (sm_100a), moments in 32 or in 8 bits.
//
// The tensors are cut into chunks, one CTA each; a table in device memory says which tensor a chunk belongs to, the
// gradients' addresses, which change from step to step, travel as arguments of the kernel.  Moments and masters lie
// in flat arrays in units of 256 values, a tensor's first value beginning a unit; a warp takes a unit.
//
// 8-bit moments: a unit's largest value gives a power of two as scale; the first moment is an e4m3 number, the second
// an e5m2 number times it.  Both are 32-bit numbers with fewer digits: with the exponent lowered by the difference of the
// types' biases the upper bits are the code, denormals included.  Rounding is stochastic, because the second moment moves by
// 1 - beta2 of its difference to g^2 per step, far less than half the distance of two e5m2 numbers, and would never
// leave its place otherwise; and scales are powers of two, because a value that has not changed is then on the new
// grid too and is not rounded again, which would add up to a noise of several times the value over 1 / (1 - beta2) steps.
// Second moments above zero stay above zero.
#include "training.h"

#include <math.h>

namespace ffcvb {

namespace {

constexpr int kUnit = FFCVB_ADAMW_BLOCK;
constexpr int kThreads = 256;
constexpr int kUnitsPerChunk = 32;
constexpr long long kChunk = (long long)kUnit * kUnitsPerChunk;
constexpr int kSets = 16; // different (group, steps) of one launch

struct Tensor {
    uint64_t param;
    int64_t numel, start;
};
struct Chunk {
    int32_t tensor, index;
};

long long chunks_of(int64_t numel) { return (numel + kChunk - 1) / kChunk; }

// What the tensors of one group that have made equally many steps share.
struct Set {
    float b1, c1, b2, c2; // c = 1 - b
    float decay, rate, over_root, eps;
    uint32_t key;
};

template <int MOST> struct Launch {
    const void *grads[MOST];
    Set sets[kSets];
    uint8_t set[MOST];
    const Tensor *tensors; // of the launch
    const Chunk *chunks;
    int first;             // tensor
    void *exp_avg, *exp_avg_sq;
    float *scales, *master;
    const float *norm;     // or NULL
    float max_norm;
    float *partial;
};

__host__ __device__ inline uint32_t mix(uint32_t x) {
    x *= 0xE4C6EF2Bu;
    x ^= x >> 15;
    x *= 0x87EA99B3u;
    return x ^ (x >> 16);
}

// Four values from place `at` of a tensor of n; 0 beyond its end.
template <typename T>
__device__ __forceinline__ void load4(float (&v)[4], const T *p, long long at, long long n, bool aligned) {
    if (aligned && at + 4 <= n) {
        if constexpr (sizeof(T) == 4) {
            const float4 f = __ldcs(reinterpret_cast<const float4 *>(p + at));
            v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
        } else {
            const uint2 w = __ldcs(reinterpret_cast<const uint2 *>(p + at));
            T t[4];
            *reinterpret_cast<uint2 *>(t) = w;
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] = to_float(t[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = at + j < n ? to_float(p[at + j]) : 0.0f;
    }
}
template <typename T>
__device__ __forceinline__ void store4(const float (&v)[4], T *p, long long at, long long n, bool aligned) {
    if (aligned && at + 4 <= n) {
        if constexpr (sizeof(T) == 4) {
            __stcs(reinterpret_cast<float4 *>(p + at), make_float4(v[0], v[1], v[2], v[3]));
        } else {
            T t[4];
#pragma unroll
            for (int j = 0; j < 4; j++) t[j] = from_float<T>(v[j]);
            __stcs(reinterpret_cast<uint2 *>(p + at), *reinterpret_cast<const uint2 *>(t));
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (at + j < n) p[at + j] = from_float<T>(v[j]);
    }
}

// 2^e as a number, -127 < e < 128.
__device__ __forceinline__ float power(int e) { return __int_as_float((e + 127) << 23); }

// Codes of eight values of a lane, and the unit's scale; the largest becomes 2^TOP .. 2^(TOP + 1).
template <int TOP, int BIAS, int DROPPED>
__device__ __forceinline__ float to_eight(const float (&v)[8], const uint32_t (&noise)[8], uint32_t (&code)[2]) {
    float most = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; j++) most = fmaxf(most, fabsf(v[j]));
    bool odd = false; // not a number: fmaxf does not see it
#pragma unroll
    for (int j = 0; j < 8; j++) odd |= v[j] != v[j];
    uint32_t top = __reduce_max_sync(0xffffffffu, odd ? 0x7fc00000u : __float_as_uint(most)) >> 23;
    if (top >= 255) {
        code[0] = code[1] = 0x01010101u;
        return NAN; // infinities and what is no number make the unit none
    }
    const int e = max((int)top, 1) - 127;
    const float down = power(-e), bias = __int_as_float((127 + TOP - BIAS) << 23);
    code[0] = code[1] = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        uint32_t c = (__float_as_uint(__fmul_rn(__fmul_rn(fabsf(v[j]), down), bias)) + noise[j]) >> DROPPED;
        if (DROPPED == 21) c = max(c, v[j] > 0.0f ? 1u : 0u);
        if (DROPPED == 20 && v[j] < 0.0f) c |= 128u;
        code[j >> 2] |= c << (8 * (j & 3));
    }
    return __fmul_rn(power(e), __int_as_float((127 - TOP) << 23));
}
template <int TOP, int BIAS, int DROPPED>
__device__ __forceinline__ float from_eight(uint32_t code, int j, float scale) {
    const uint32_t c = code >> (8 * j);
    const float v = __int_as_float((c & 127u) << DROPPED | (c & 128u) << 24);
    return __fmul_rn(__fmul_rn(v, __int_as_float((127 + BIAS) << 23)), scale);
}

template <typename T, int BITS, int MOST>
__global__ void __launch_bounds__(kThreads)
step_kernel(const __grid_constant__ Launch<MOST> a) {
    const Chunk chunk = a.chunks[blockIdx.x];
    const int local = chunk.tensor - a.first;
    const T *grad = static_cast<const T *>(a.grads[local]);
    if (!grad) return;
    float clip = 1.0f;
    if (a.norm) {
        const float norm = *a.norm;
        if (!isfinite(norm)) return;
        clip = fminf(1.0f, a.max_norm / (norm + 1e-6f));
    }
    const Tensor tensor = a.tensors[local];
    const Set set = a.sets[a.set[local]];
    T *param = reinterpret_cast<T *>(tensor.param);
    const long long n = tensor.numel;
    const bool aligned = ((reinterpret_cast<uintptr_t>(grad) | reinterpret_cast<uintptr_t>(param)) & (4 * sizeof(T) - 1)) == 0;
    const int lane = threadIdx.x & 31;
    for (int unit = threadIdx.x >> 5; unit < kUnitsPerChunk; unit += kThreads / 32) {
        const long long first = chunk.index * kChunk + unit * kUnit; // in the tensor
        if (first >= n) break;
        const long long flat = tensor.start + first;
        float g[8], w[8], m[8], v[8];
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const long long at = first + half * 128 + lane * 4;
            const long long place = flat + half * 128 + lane * 4;
            float(&g4)[4] = *reinterpret_cast<float(*)[4]>(g + 4 * half);
            float(&w4)[4] = *reinterpret_cast<float(*)[4]>(w + 4 * half);
            load4(g4, grad, at, n, aligned);
            if (sizeof(T) == 4)
                load4(w4, param, at, n, aligned);
            else
                *reinterpret_cast<float4 *>(w4) = __ldcs(reinterpret_cast<const float4 *>(a.master + place));
            if (BITS == 32) {
                *reinterpret_cast<float4 *>(m + 4 * half) = __ldcs(reinterpret_cast<const float4 *>(static_cast<const float *>(a.exp_avg) + place));
                *reinterpret_cast<float4 *>(v + 4 * half) = __ldcs(reinterpret_cast<const float4 *>(static_cast<const float *>(a.exp_avg_sq) + place));
            } else {
                const float2 scale = *reinterpret_cast<const float2 *>(a.scales + flat / kUnit * 2);
                const uint32_t mc = __ldcs(reinterpret_cast<const uint32_t *>(static_cast<const uint8_t *>(a.exp_avg) + place));
                const uint32_t vc = __ldcs(reinterpret_cast<const uint32_t *>(static_cast<const uint8_t *>(a.exp_avg_sq) + place));
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    m[4 * half + j] = from_eight<7, 120, 20>(mc, j, scale.x);
                    v[4 * half + j] = from_eight<14, 112, 21>(vc, j, scale.y);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float gj = __fmul_rn(g[j], clip);
            m[j] = __fadd_rn(__fmul_rn(m[j], set.b1), __fmul_rn(gj, set.c1));
            v[j] = __fadd_rn(__fmul_rn(v[j], set.b2), __fmul_rn(__fmul_rn(gj, gj), set.c2));
            w[j] = w[j] * set.decay - set.rate * (m[j] / (sqrtf(v[j]) * set.over_root + set.eps));
        }
        uint32_t mc[2], vc[2];
        if (BITS == 8) {
            const uint32_t base = (uint32_t)flat + set.key + (uint32_t)(flat >> 32) * 0x9E3779B9u;
            uint32_t m_noise[8], v_noise[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const uint32_t r = mix(base + (j >> 2) * 128 + lane * 4 + (j & 3));
                m_noise[j] = (r & 0xffffu) << 4;
                v_noise[j] = (r >> 16) << 5;
            }
            float2 scale;
            scale.x = to_eight<7, 120, 20>(m, m_noise, mc);
            scale.y = to_eight<14, 112, 21>(v, v_noise, vc);
            if (lane == 0) *reinterpret_cast<float2 *>(a.scales + flat / kUnit * 2) = scale;
        }
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const long long at = first + half * 128 + lane * 4;
            const long long place = flat + half * 128 + lane * 4;
            const float(&w4)[4] = *reinterpret_cast<const float(*)[4]>(w + 4 * half);
            store4(w4, param, at, n, aligned);
            if (sizeof(T) != 4) __stcs(reinterpret_cast<float4 *>(a.master + place), make_float4(w4[0], w4[1], w4[2], w4[3]));
            if (BITS == 32) {
                __stcs(reinterpret_cast<float4 *>(static_cast<float *>(a.exp_avg) + place), make_float4(m[4 * half], m[4 * half + 1], m[4 * half + 2], m[4 * half + 3]));
                __stcs(reinterpret_cast<float4 *>(static_cast<float *>(a.exp_avg_sq) + place), make_float4(v[4 * half], v[4 * half + 1], v[4 * half + 2], v[4 * half + 3]));
            } else {
                __stcs(reinterpret_cast<uint32_t *>(static_cast<uint8_t *>(a.exp_avg) + place), mc[half]);
                __stcs(reinterpret_cast<uint32_t *>(static_cast<uint8_t *>(a.exp_avg_sq) + place), vc[half]);
            }
        }
    }
}

// The sum of squares of a chunk's gradients.
template <typename T, int MOST>
__global__ void __launch_bounds__(kThreads)
squares_kernel(const __grid_constant__ Launch<MOST> a) {
    __shared__ float s_part[kThreads / 32];
    const Chunk chunk = a.chunks[blockIdx.x];
    const int local = chunk.tensor - a.first;
    const T *grad = static_cast<const T *>(a.grads[local]);
    float sum = 0.0f;
    if (grad) {
        const long long n = a.tensors[local].numel;
        const bool aligned = (reinterpret_cast<uintptr_t>(grad) & (4 * sizeof(T) - 1)) == 0;
        const long long first = chunk.index * kChunk;
        for (int k = threadIdx.x; k < kChunk / 4 && first + k * 4 < n; k += kThreads) {
            float g[4];
            load4(g, grad, first + k * 4, n, aligned);
#pragma unroll
            for (int j = 0; j < 4; j++) sum += g[j] * g[j];
        }
    }
    sum = warp_sum(sum);
    if ((threadIdx.x & 31) == 0) s_part[threadIdx.x >> 5] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
        for (int k = 1; k < kThreads / 32; k++) sum += s_part[k];
        a.partial[blockIdx.x] = sum;
    }
}
__global__ void __launch_bounds__(1024)
norm_kernel(const float *__restrict__ partial, long long n, float *norm) {
    __shared__ double s_sum[32];
    double sum = 0.0;
    for (long long k = threadIdx.x; k < n; k += 1024) sum += partial[k];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if ((threadIdx.x & 31) == 0) s_sum[threadIdx.x >> 5] = sum;
    __syncthreads();
    if (threadIdx.x < 32) {
        sum = s_sum[threadIdx.x];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (threadIdx.x == 0) *norm = (float)sqrt(sum);
    }
}

struct Tensors { // HOST
    const int64_t *numel;
    const uint64_t *grads;
    const int64_t *steps;
    const int32_t *group_of;
    const ffcvb_adamw_group *groups;
    long long chunks;
};

// Every launch takes as many tensors as its arguments have room for.
template <typename T, int MOST>
void launch_all(const ffcvb_adamw_args &args, const Tensors &t, bool squares, cudaStream_t st) {
    const Tensor *tensors = static_cast<const Tensor *>(args.tensors);
    const Chunk *chunks = reinterpret_cast<const Chunk *>(tensors + args.n_tensors);
    long long at = 0; // chunk
    for (int first = 0; first < args.n_tensors;) {
        Launch<MOST> a;
        int sets = 0, n = 0, group[kSets];
        int64_t steps[kSets];
        long long count = 0;
        bool any = false;
        for (; n < MOST && first + n < args.n_tensors; n++) {
            const int i = first + n;
            a.grads[n] = reinterpret_cast<const void *>(t.grads[i]);
            a.set[n] = 0;
            if (a.grads[n] && !squares) {
                int s = 0;
                while (s < sets && (group[s] != t.group_of[i] || steps[s] != t.steps[i])) s++;
                if (s == sets) {
                    if (sets == kSets) break;
                    const ffcvb_adamw_group &g = t.groups[t.group_of[i]];
                    const double step = (double)t.steps[i];
                    group[s] = t.group_of[i];
                    steps[s] = t.steps[i];
                    Set &to = a.sets[sets++];
                    to.b1 = (float)g.beta1;
                    to.c1 = (float)(1.0 - g.beta1);
                    to.b2 = (float)g.beta2;
                    to.c2 = (float)(1.0 - g.beta2);
                    to.decay = (float)(1.0 - g.lr * g.weight_decay);
                    to.rate = (float)(g.lr / (1.0 - pow(g.beta1, step)));
                    to.over_root = (float)(1.0 / sqrt(1.0 - pow(g.beta2, step)));
                    to.eps = (float)g.eps;
                    to.key = mix(mix((uint32_t)args.seed + 1u) ^ (uint32_t)t.steps[i]);
                }
                a.set[n] = (uint8_t)s;
            }
            any |= a.grads[n] != nullptr;
            count += chunks_of(t.numel[i]);
        }
        a.tensors = tensors + first;
        a.chunks = chunks + at;
        a.first = first;
        a.exp_avg = args.exp_avg;
        a.exp_avg_sq = args.exp_avg_sq;
        a.scales = args.scales;
        a.master = args.master;
        a.norm = args.max_norm > 0.0 ? args.norm : nullptr;
        a.max_norm = (float)args.max_norm;
        a.partial = static_cast<float *>(args.workspace) + at;
        if (count > 0 && (any || squares)) {
            if (squares)
                squares_kernel<T, MOST><<<(unsigned)count, kThreads, 0, st>>>(a);
            else if (args.bits == 8)
                step_kernel<T, 8, MOST><<<(unsigned)count, kThreads, 0, st>>>(a);
            else
                step_kernel<T, 32, MOST><<<(unsigned)count, kThreads, 0, st>>>(a);
        }
        first += n;
        at += count;
    }
}

} // namespace

} // namespace ffcvb

using namespace ffcvb;

extern "C" {

int64_t ffcvb_adamw_layout(int32_t n, const int64_t *numel, int64_t *start, int64_t *sizes) {
    int64_t at = 0, chunks = 0;
    for (int32_t i = 0; i < n; i++) {
        start[i] = at;
        at += (numel[i] + kUnit - 1) / kUnit * kUnit;
        chunks += chunks_of(numel[i]);
    }
    sizes[0] = n * (int64_t)sizeof(Tensor) + chunks * (int64_t)sizeof(Chunk);
    sizes[1] = chunks * (int64_t)sizeof(float);
    return at;
}

int ffcvb_adamw_table(int32_t n, const int64_t *numel, const uint64_t *params, void *table) {
    if (n < 0 || (n > 0 && (!numel || !params || !table))) return training_fail(FFCVB_E_ARG, "ffcvb_adamw_table: bad argument");
    Tensor *tensors = static_cast<Tensor *>(table);
    Chunk *chunk = reinterpret_cast<Chunk *>(tensors + n);
    int64_t at = 0;
    for (int32_t i = 0; i < n; i++) {
        if (chunks_of(numel[i]) > 0x7fffffff) return training_fail(FFCVB_E_LIMIT, "ffcvb_adamw_table: tensor %d is too large", i);
        tensors[i] = Tensor{params[i], numel[i], at};
        at += (numel[i] + kUnit - 1) / kUnit * kUnit;
        for (int64_t c = 0; c < chunks_of(numel[i]); c++) *chunk++ = Chunk{i, (int32_t)c};
    }
    return FFCVB_OK;
}

int ffcvb_adamw_step(const ffcvb_adamw_args *args, const int64_t *numel, const uint64_t *grads, int64_t *steps,
                     const int32_t *group_of, const ffcvb_adamw_group *groups, int32_t n_groups, void *stream) {
    if (!args || args->n_tensors < 0) return training_fail(FFCVB_E_ARG, "ffcvb_adamw_step: no arguments");
    const ffcvb_adamw_args &a = *args;
    if (a.n_tensors == 0) return FFCVB_OK;
    if (!numel || !grads || !steps || !group_of || !groups || !a.tensors || !a.exp_avg || !a.exp_avg_sq || (a.bits != 8 && a.bits != 32) ||
        (a.bits == 8 && !a.scales) || (a.type != FFCVB_TYPE_F32 && (!a.master || (a.type != FFCVB_TYPE_F16 && a.type != FFCVB_TYPE_BF16))) ||
        (a.max_norm > 0.0 && (!a.norm || !a.workspace)))
        return training_fail(FFCVB_E_ARG, "ffcvb_adamw_step: bad argument");
    Tensors t{numel, grads, steps, group_of, groups, 0};
    for (int32_t i = 0; i < a.n_tensors; i++) {
        if (group_of[i] < 0 || group_of[i] >= n_groups) return training_fail(FFCVB_E_ARG, "ffcvb_adamw_step: tensor %d is in no group", i);
        t.chunks += chunks_of(numel[i]);
    }
    if (t.chunks > 0x7fffffff) return training_fail(FFCVB_E_LIMIT, "ffcvb_adamw_step: too many values");
    OnDevice here(a.device);
    if (!here.ok()) return training_fail(FFCVB_E_NODEVICE, "ffcvb_adamw_step: no device %d", a.device);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    for (int32_t i = 0; i < a.n_tensors; i++) steps[i] += grads[i] != 0;
    with_type(a.type, [&](auto zero) {
        using T = decltype(zero);
        auto all = [&](bool squares) {
            if (a.n_tensors <= 64)
                launch_all<T, 64>(a, t, squares, st);
            else
                launch_all<T, 1024>(a, t, squares, st);
        };
        if (a.max_norm > 0.0) {
            all(true);
            norm_kernel<<<1, 1024, 0, st>>>(static_cast<const float *>(a.workspace), t.chunks, a.norm);
        }
        all(false);
    });
    return launched("ffcvb_adamw_step");
}

} // extern "C"
