// One AdamW step over many tensors (sm_100a), moments in 32 or in 8 bits.
//
// The tensors are cut into chunks; a table in device memory says which tensor a chunk belongs to, the
// gradients' addresses, which change from step to step, travel as arguments of the kernel.  Moments and masters lie
// in flat arrays in units of 256 values, a tensor's first value beginning a unit; a warp takes a unit.
//
// 8-bit moments: a unit's largest value gives a power of two as scale; the first moment is an e4m3 number, the second
// an e5m2 number times it.  Both are 32-bit numbers with fewer digits: with the exponent lowered by the difference of the
// types' biases the upper bits are the code, denormals included.  Rounding is stochastic, because the second moment moves by
// 1 - beta2 of its difference to g^2 per step, far less than half the distance of two e5m2 numbers, and would never
// leave its place otherwise; and scales are powers of two, because a value that has not changed is then on the new
// grid too and is not rounded again, which would add up to a noise of several times the value over 1 / (1 - beta2) steps.
// A second moment above zero keeps the smallest code at least, except below 2^-128.
//
// Reading and writing bounds it: 28 bytes per value with moments in 32 bits, with 8-bit moments 16, masters of 16-bit weights included.
// 409 M bf16 weights with 8-bit moments: 981 us (1002 at the rate of a copy); 101 M values in 32 bits with clipping, which reads the
// gradients twice: 477 us (492 at that rate, had the caches kept nothing).
#include "training.h"
#include "two.h"

#include <math.h>
#include <type_traits>

namespace ffcvb {

namespace {

constexpr int kUnit = FFCVB_ADAMW_BLOCK;
constexpr int kThreads = 256;
constexpr int kPlaces = 4; // CTAs of an SM in a step with 8-bit moments
constexpr int kSets = 16; // different (group, steps) of one launch

struct Tensor {
    uint64_t param;
    int64_t numel, start;
};
struct Chunk {
    int32_t tensor, index;
};

// Values of a chunk, of which the squares' kernel gives one to a CTA: with a chunk for every second SM four loads of 16 bytes a thread are
// in flight at once instead of one (25 M values, squares and step: 124 us, 136 with short ones; 850 000: 8.8, 9.8); with fewer, short ones
// bring more SMs in (500 000: 8.7 us, 9.1 with long ones; 51 000: 7.2, 8.0).
constexpr long long kShort = 8 * kUnit, kLong = 32 * kUnit;
long long chunk_size(int32_t n, const int64_t *numel) {
    int64_t all = 0;
    for (int32_t i = 0; i < n; i++) all += numel[i];
    return all < kSms / 2 * kLong ? kShort : kLong;
}
long long chunks_of(int64_t numel, long long chunk) { return (numel + chunk - 1) / chunk; }

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
    int chunk;             // values
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

// Four neighbouring values as two pairs.
__device__ __forceinline__ void four(Two *v, float4 f) {
    v[0] = Two(f.x, f.y);
    v[1] = Two(f.z, f.w);
}
__device__ __forceinline__ float4 four(const Two *v) { return make_float4(v[0].lo(), v[0].hi(), v[1].lo(), v[1].hi()); }

// Four values as they lie in memory.
template <typename T> struct Words {
    uint2 v;
    __device__ __forceinline__ float4 get() const {
        float2 lo, hi;
        if constexpr (std::is_same<T, __half>::value) {
            lo = __half22float2(*reinterpret_cast<const __half2 *>(&v.x));
            hi = __half22float2(*reinterpret_cast<const __half2 *>(&v.y));
        } else {
            lo = make_float2(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u));
            hi = make_float2(__uint_as_float(v.y << 16), __uint_as_float(v.y & 0xffff0000u));
        }
        return make_float4(lo.x, lo.y, hi.x, hi.y);
    }
};
template <> struct Words<float> {
    float4 v;
    __device__ __forceinline__ float4 get() const { return v; }
};
// Those from place `at` of a tensor of n; 0 beyond its end.  WHOLE: none is, and the tensor lies on boundaries of four values.
template <bool WHOLE, typename T>
__device__ __forceinline__ Words<T> load4(const T *p, long long at, long long n) {
    if constexpr (WHOLE) {
        return *reinterpret_cast<const Words<T> *>(p + at);
    } else if constexpr (sizeof(T) == 4) {
        return {make_float4(at < n ? p[at] : 0.0f, at + 1 < n ? p[at + 1] : 0.0f, at + 2 < n ? p[at + 2] : 0.0f, at + 3 < n ? p[at + 3] : 0.0f)};
    } else {
        const uint16_t *q = reinterpret_cast<const uint16_t *>(p);
        const uint32_t v0 = at < n ? q[at] : 0, v1 = at + 1 < n ? q[at + 1] : 0, v2 = at + 2 < n ? q[at + 2] : 0, v3 = at + 3 < n ? q[at + 3] : 0;
        return {make_uint2(v0 | v1 << 16, v2 | v3 << 16)};
    }
}
template <bool WHOLE, typename T>
__device__ __forceinline__ void store4(float4 v, T *p, long long at, long long n) {
    if constexpr (WHOLE && sizeof(T) == 4) {
        *reinterpret_cast<float4 *>(p + at) = v;
    } else if constexpr (WHOLE) {
        uint2 w;
        if constexpr (std::is_same<T, __half>::value) {
            const __half2 lo = __floats2half2_rn(v.x, v.y), hi = __floats2half2_rn(v.z, v.w);
            w = make_uint2(*reinterpret_cast<const uint32_t *>(&lo), *reinterpret_cast<const uint32_t *>(&hi));
        } else {
            const __nv_bfloat162 lo = __floats2bfloat162_rn(v.x, v.y), hi = __floats2bfloat162_rn(v.z, v.w);
            w = make_uint2(*reinterpret_cast<const uint32_t *>(&lo), *reinterpret_cast<const uint32_t *>(&hi));
        }
        *reinterpret_cast<uint2 *>(p + at) = w;
    } else {
        if (at < n) p[at] = from_float<T>(v.x);
        if (at + 1 < n) p[at + 1] = from_float<T>(v.y);
        if (at + 2 < n) p[at + 2] = from_float<T>(v.z);
        if (at + 3 < n) p[at + 3] = from_float<T>(v.w);
    }
}

// 2^e as a number, -127 < e < 128.
__device__ __forceinline__ float power(int e) { return __int_as_float((e + 127) << 23); }

// The largest of three sizes; what is no number is larger.
__device__ __forceinline__ float largest(float a, float b, float c) {
    float r;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// The unit's scale for eight values of every lane, of which the largest becomes 2^TOP .. 2^(TOP + 1); v becomes the 32-bit numbers
// that have an 8-bit type's codes as their upper bits.  Infinities and what is no number make the unit none.
template <int TOP, int BIAS>
__device__ __forceinline__ float scale_down(Two (&v)[4]) {
    float most = largest(v[0].lo(), v[0].hi(), v[1].lo());
    most = largest(most, v[1].hi(), v[2].lo());
    most = largest(most, v[2].hi(), v[3].lo());
    most = largest(most, v[3].hi(), 0.0f);
    const int e = max((int)(__reduce_max_sync(0xffffffffu, __float_as_uint(most)) >> 23), 1) - 127;
    const float down = e < 128 ? power(-e) : 0.0f, bias = __int_as_float((127 + TOP - BIAS) << 23);
#pragma unroll
    for (int p = 0; p < 4; p++) v[p] = mul_rn(mul_rn(v[p], Two(down, down)), Two(bias, bias));
    return e < 128 ? __fmul_rn(power(e), __int_as_float((127 - TOP) << 23)) : NAN;
}
// The upper bytes of four words, the first lowest.
__device__ __forceinline__ uint32_t top_bytes(const uint32_t *w) {
    return __byte_perm(__byte_perm(w[0], w[1], 0x0073), __byte_perm(w[2], w[3], 0x0073), 0x5410);
}

// What a lane reads of a unit: four neighbours in either half of it.  WHOLE: all of it inside a tensor on boundaries of four values.
template <typename T, int BITS> struct Unit {
    Words<T> g[2];
    float4 w[2], m[BITS == 32 ? 2 : 1], v[BITS == 32 ? 2 : 1];
    uint32_t mc[2], vc[2];
    float2 scale;
    template <bool WHOLE, typename Args>
    __device__ __forceinline__ void load(const Args &a, const T *grad, const T *param, long long first, long long n, long long flat) {
        const int lane = threadIdx.x & 31;
        if (BITS == 8) scale = *reinterpret_cast<const float2 *>(a.scales + flat / kUnit * 2);
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const long long at = first + half * 128 + lane * 4, place = flat + half * 128 + lane * 4;
            g[half] = load4<WHOLE>(grad, at, n);
            if constexpr (sizeof(T) == 4)
                w[half] = load4<WHOLE>(param, at, n).v;
            else
                w[half] = *reinterpret_cast<const float4 *>(a.master + place);
            if constexpr (BITS == 32) {
                m[half] = *reinterpret_cast<const float4 *>(static_cast<const float *>(a.exp_avg) + place);
                v[half] = *reinterpret_cast<const float4 *>(static_cast<const float *>(a.exp_avg_sq) + place);
            } else {
                mc[half] = static_cast<const uint32_t *>(a.exp_avg)[place / 4];
                vc[half] = static_cast<const uint32_t *>(a.exp_avg_sq)[place / 4];
            }
        }
    }
};

template <typename T, int BITS, bool WHOLE, typename Args>
__device__ __forceinline__ void step_unit(const Args &a, const Unit<T, BITS> &unit, const Set &set, float clip, T *param, long long first, long long n, long long flat) {
    const int lane = threadIdx.x & 31;
    Two g[4], w[4], m[4], v[4];
    float *const exp_avg = static_cast<float *>(a.exp_avg), *const exp_avg_sq = static_cast<float *>(a.exp_avg_sq);
    uint32_t *const m_codes = static_cast<uint32_t *>(a.exp_avg), *const v_codes = static_cast<uint32_t *>(a.exp_avg_sq);
    uint32_t mc[2], vc[2];
    float2 scale = unit.scale;
#pragma unroll
    for (int half = 0; half < 2; half++) {
        four(g + 2 * half, unit.g[half].get());
        four(w + 2 * half, unit.w[half]);
        if constexpr (BITS == 32) {
            four(m + 2 * half, unit.m[half]);
            four(v + 2 * half, unit.v[half]);
        } else {
            mc[half] = unit.mc[half];
            vc[half] = unit.vc[half];
        }
    }
    if (BITS == 8) {
#pragma unroll
        for (int p = 0; p < 4; p++) { // through 16-bit floats, which hold either type: e5m2 numbers are their upper bytes
            const uint32_t two_m = mc[p >> 1] >> (16 * (p & 1));
            uint32_t halves;
            asm("{ .reg .b16 c; cvt.u16.u32 c, %1; cvt.rn.f16x2.e4m3x2 %0, c; }" : "=r"(halves) : "r"(two_m));
            const float2 fm = __half22float2(*reinterpret_cast<const __half2 *>(&halves));
            m[p] = mul_rn(Two(fm.x, fm.y), Two(scale.x, scale.x));
            halves = __byte_perm(vc[p >> 1], 0, p & 1 ? 0x3424 : 0x1404);
            const float2 fv = __half22float2(*reinterpret_cast<const __half2 *>(&halves));
            v[p] = mul_rn(Two(fv.x, fv.y), Two(scale.y, scale.y));
        }
    }
    const Two c2(clip, clip), b1(set.b1, set.b1), d1(set.c1, set.c1), b2(set.b2, set.b2), d2(set.c2, set.c2);
#pragma unroll
    for (int p = 0; p < 4; p++) {
        g[p] = mul_rn(g[p], c2);
        m[p] = add_rn(mul_rn(m[p], b1), mul_rn(g[p], d1));
        v[p] = add_rn(mul_rn(v[p], b2), mul_rn(mul_rn(g[p], g[p]), d2));
        // (a root and a quotient to within two units of the last place: they change a weight by a thousandth of its size at most)
        float root[2], u[2];
#pragma unroll
        for (int j = 0; j < 2; j++) {
            asm("sqrt.approx.f32 %0, %1;" : "=f"(root[j]) : "f"(v[p].half(j)));
            asm("div.approx.ftz.f32 %0, %1, %2;" : "=f"(u[j]) : "f"(m[p].half(j)), "f"(fmaf(root[j], set.over_root, set.eps)));
        }
        w[p] = fma_rn(Two(u[0], u[1]), Two(-set.rate, -set.rate), mul_rn(w[p], Two(set.decay, set.decay)));
    }
    if (BITS == 8) {
        uint32_t lifted[4]; // (v's smallest code: above zero; values below 2^-128 may still become zero)
        scale.x = scale_down<7, 120>(m);
        Two down[4] = {v[0], v[1], v[2], v[3]};
        scale.y = scale_down<14, 112>(down);
        const uint32_t base = ((uint32_t)flat + set.key + (uint32_t)(flat >> 32) * 0x9E3779B9u + lane * 4) * 0xE4C6EF2Bu;
#pragma unroll
        for (int half = 0; half < 2; half++) {
            uint32_t m_word[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                uint32_t x = base + (half * 128 + j) * 0xE4C6EF2Bu; // mix(place + key)
                x ^= x >> 15;
                x *= 0x87EA99B3u;
                const uint32_t upper = x >> 16;
                const uint32_t y = __float_as_uint(m[2 * half + (j >> 1)].half(j & 1)) + (((x ^ upper) & 0xffffu) << 4);
                m_word[j] = (y & 0x80000000u) | ((y << 4) & 0x7fffffffu);
                uint32_t z = __float_as_uint(down[2 * half + (j >> 1)].half(j & 1)) + (upper << 5);
                z = max(z, min(__float_as_uint(v[2 * half + (j >> 1)].half(j & 1)), 1u << 21));
                lifted[j] = z << 3;
            }
            mc[half] = top_bytes(m_word);
            vc[half] = top_bytes(lifted);
        }
        if (lane == 0) *reinterpret_cast<float2 *>(a.scales + flat / kUnit * 2) = scale;
    }
#pragma unroll
    for (int half = 0; half < 2; half++) {
        const long long at = first + half * 128 + lane * 4, place = flat + half * 128 + lane * 4;
        store4<WHOLE>(four(w + 2 * half), param, at, n);
        if (sizeof(T) != 4) *reinterpret_cast<float4 *>(a.master + place) = four(w + 2 * half);
        if (BITS == 32) {
            *reinterpret_cast<float4 *>(exp_avg + place) = four(m + 2 * half);
            *reinterpret_cast<float4 *>(exp_avg_sq + place) = four(v + 2 * half);
        } else {
            m_codes[place / 4] = mc[half];
            v_codes[place / 4] = vc[half];
        }
    }
}

// A whole unit on its way through a warp's part of shared memory.
template <typename T> struct alignas(16) Staged {
    T g[kUnit];
    float w[kUnit];
    uint32_t mc[kUnit / 4], vc[kUnit / 4];
    float2 scale[2];
    template <int BYTES>
    static __device__ __forceinline__ void copy(void *to, const void *from) {
        const uint32_t at = (uint32_t)__cvta_generic_to_shared(to);
        if constexpr (BYTES == 16)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(from) : "memory");
        else
            asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(at), "l"(from) : "memory");
    }
    template <typename Args>
    __device__ __forceinline__ void begin(const Args &a, const T *grad, const T *param, long long first, long long flat) {
        const int lane = threadIdx.x & 31, codes = (lane & 15) * 4;
        const float *from;
        if constexpr (sizeof(T) == 4)
            from = param + first;
        else
            from = a.master + flat;
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const int at = half * 128 + lane * 4;
            copy<4 * sizeof(T)>(g + at, grad + first + at);
            copy<16>(w + at, from + at);
        }
        copy<16>((lane < 16 ? mc : vc) + codes, static_cast<const uint32_t *>(lane < 16 ? a.exp_avg : a.exp_avg_sq) + flat / 4 + codes);
        if (lane == 0) copy<8>(scale, a.scales + flat / kUnit * 2);
    }
    __device__ __forceinline__ void read(Unit<T, 8> &u) const {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const int at = half * 128 + lane * 4;
            u.g[half] = *reinterpret_cast<const Words<T> *>(g + at);
            u.w[half] = *reinterpret_cast<const float4 *>(w + at);
            u.mc[half] = mc[at / 4];
            u.vc[half] = vc[at / 4];
        }
        u.scale = scale[0];
    }
};

// STAGED: a CTA takes a whole chunk, with the next unit's copies under way while a warp works on one.  Otherwise it takes kShort values,
// a warp a unit: in 32 bits, where the work is little, that keeps memory as busy (101 M bf16 values and their squares: 477 us).  With
// 8-bit moments a warp that waits for each unit's loads leaves memory idle while it works: 409 M bf16 values take 981 us staged, 1143
// without, 1114 with the next unit in registers, of which three CTAs fit instead of four.
template <typename T, int BITS, int MOST, bool STAGED>
__global__ void __launch_bounds__(kThreads, BITS == 8 ? kPlaces : 1)
step_kernel(const __grid_constant__ Launch<MOST> a) {
    wait_for_previous();
    let_next_begin();
    const unsigned parts = STAGED ? 1 : (unsigned)a.chunk / (unsigned)kShort;
    const Chunk chunk = a.chunks[blockIdx.x / parts];
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
    const Set &set = a.sets[a.set[local]];
    T *param = reinterpret_cast<T *>(tensor.param);
    const long long n = tensor.numel;
    const bool aligned = ((reinterpret_cast<uintptr_t>(grad) | reinterpret_cast<uintptr_t>(param)) & (4 * sizeof(T) - 1)) == 0;
    long long first = (long long)chunk.index * a.chunk + (blockIdx.x % parts) * kShort + (threadIdx.x >> 5) * kUnit; // in the tensor
    Unit<T, BITS> unit;
    if constexpr (STAGED) {
        __shared__ Staged<T> s_staged[kThreads / 32][2];
        Staged<T> *const mine = s_staged[threadIdx.x >> 5];
        const long long end = min(n, (long long)(chunk.index + 1) * a.chunk);
        auto whole = [&](long long at) { return aligned && at + kUnit <= end; };
        auto begin = [&](int turn, long long at) {
            if (whole(at)) mine[turn].begin(a, grad, param, at, tensor.start + at);
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        begin(0, first);
        for (int turn = 0; whole(first); first += kShort, turn ^= 1) {
            __syncwarp(); // (all lanes have read what the next copies overwrite)
            begin(turn ^ 1, first + kShort);
            asm volatile("cp.async.wait_group 1;" ::: "memory");
            __syncwarp();
            mine[turn].read(unit);
            step_unit<T, BITS, true>(a, unit, set, clip, param, first, n, tensor.start + first);
        }
        for (; first < end; first += kShort) {
            unit.template load<false>(a, grad, param, first, n, tensor.start + first);
            step_unit<T, BITS, false>(a, unit, set, clip, param, first, n, tensor.start + first);
        }
    } else {
        if (first >= n) return;
        if (aligned && first + kUnit <= n) {
            unit.template load<true>(a, grad, param, first, n, tensor.start + first);
            step_unit<T, BITS, true>(a, unit, set, clip, param, first, n, tensor.start + first);
        } else {
            unit.template load<false>(a, grad, param, first, n, tensor.start + first);
            step_unit<T, BITS, false>(a, unit, set, clip, param, first, n, tensor.start + first);
        }
    }
}
// With 8-bit moments, where there is a long chunk for each place of a CTA: 6.5 M values take 21.5 us staged, 24.4 without; 1.1 M take
// 10.3 and 5.8, as a CTA's four units are one after another.
bool staged(int bits, long long values) { return bits == 8 && values >= kSms * kPlaces * kLong; }

// The sum of squares of a chunk's gradients.  The last chunks come first: what the first ones leave in the caches the step begins with
// (101 M values in 32 bits, in a step of 505 us: 3 us less than with the first chunks first).
template <typename T, int MOST>
__global__ void __launch_bounds__(kThreads)
squares_kernel(const __grid_constant__ Launch<MOST> a) {
    __shared__ float s_part[kThreads / 32];
    wait_for_previous();
    let_next_begin();
    const unsigned which = gridDim.x - 1 - blockIdx.x;
    const Chunk chunk = a.chunks[which];
    const int local = chunk.tensor - a.first;
    const T *grad = static_cast<const T *>(a.grads[local]);
    float sum = 0.0f;
    if (grad) {
        const long long n = a.tensors[local].numel;
        const bool aligned = (reinterpret_cast<uintptr_t>(grad) & (4 * sizeof(T) - 1)) == 0;
        const long long first = (long long)chunk.index * a.chunk;
        constexpr int AT_ONCE = kLong / 4 / kThreads;
        if (aligned && first + a.chunk <= n && a.chunk == kLong) {
            Words<T> w[AT_ONCE];
#pragma unroll
            for (int k = 0; k < AT_ONCE; k++) w[k] = load4<true>(grad, first + (k * kThreads + threadIdx.x) * 4, n);
#pragma unroll
            for (int k = 0; k < AT_ONCE; k++) {
                const float4 g = w[k].get();
                sum += (g.x * g.x + g.y * g.y) + (g.z * g.z + g.w * g.w);
            }
        } else {
            for (int k = threadIdx.x; k < a.chunk / 4 && first + k * 4 < n; k += kThreads) {
                const float4 g = load4<false>(grad, first + k * 4, n).get();
                sum += (g.x * g.x + g.y * g.y) + (g.z * g.z + g.w * g.w);
            }
        }
    }
    sum = warp_sum(sum);
    if ((threadIdx.x & 31) == 0) s_part[threadIdx.x >> 5] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
        for (int k = 1; k < kThreads / 32; k++) sum += s_part[k];
        a.partial[which] = sum;
    }
}
// Masters of a chunk's weights that have been written to: where a weight is not its master rounded, it becomes the master.  A tensor's
// place in the gradients is not 0 where it is to be looked at.  (290 tensors, 408 M bf16 values: 357 us, 374 at the rate
// of a copy; the check of a loaded state by elementwise operations took 9.5 ms.)
template <typename T, int MOST>
__global__ void __launch_bounds__(kThreads)
masters_kernel(const __grid_constant__ Launch<MOST> a) {
    wait_for_previous();
    let_next_begin();
    const Chunk chunk = a.chunks[blockIdx.x];
    const int local = chunk.tensor - a.first;
    if (!a.grads[local]) return;
    const Tensor tensor = a.tensors[local];
    const T *param = reinterpret_cast<const T *>(tensor.param);
    float *const master = a.master + tensor.start;
    const long long n = tensor.numel, first = (long long)chunk.index * a.chunk;
    const bool whole = (reinterpret_cast<uintptr_t>(param) & (4 * sizeof(T) - 1)) == 0 && first + a.chunk <= n;
    for (int k = threadIdx.x; k < a.chunk / 4 && first + k * 4 < n; k += kThreads) {
        const long long at = first + k * 4;
        const float4 w = (whole ? load4<true>(param, at, n) : load4<false>(param, at, n)).get();
        float4 m = *reinterpret_cast<const float4 *>(master + at); // (behind a tensor's last value both are 0)
        auto keeps = [](float own, float weight) { return to_float(from_float<T>(own)) == weight; };
        if (keeps(m.x, w.x) && keeps(m.y, w.y) && keeps(m.z, w.z) && keeps(m.w, w.w)) continue;
        if (!keeps(m.x, w.x)) m.x = w.x;
        if (!keeps(m.y, w.y)) m.y = w.y;
        if (!keeps(m.z, w.z)) m.z = w.z;
        if (!keeps(m.w, w.w)) m.w = w.w;
        *reinterpret_cast<float4 *>(master + at) = m;
    }
}

__global__ void __launch_bounds__(1024)
norm_kernel(const float *__restrict__ partial, long long n, float *norm) {
    __shared__ double s_sum[32];
    wait_for_previous();
    let_next_begin();
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
    long long values, chunks, chunk; // of all, and values of one chunk
};

enum Pass { kSquares, kStep, kMasters };

// Every launch takes as many tensors as its arguments have room for.
template <typename T, int MOST>
void launch_all(const ffcvb_adamw_args &args, const Tensors &t, Pass pass, cudaStream_t st) {
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
            if (a.grads[n] && pass == kStep) {
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
            count += chunks_of(t.numel[i], t.chunk);
        }
        a.tensors = tensors + first;
        a.chunks = chunks + at;
        a.first = first;
        a.chunk = (int)t.chunk;
        a.exp_avg = args.exp_avg;
        a.exp_avg_sq = args.exp_avg_sq;
        a.scales = args.scales;
        a.master = args.master;
        a.norm = args.max_norm > 0.0 ? args.norm : nullptr;
        a.max_norm = (float)args.max_norm;
        a.partial = static_cast<float *>(args.workspace) + at;
        if (count > 0 && (any || pass == kSquares)) {
            const bool whole_chunks = pass != kStep || staged(args.bits, t.values);
            auto step = args.bits == 32 ? step_kernel<T, 32, MOST, false> : whole_chunks ? step_kernel<T, 8, MOST, true> : step_kernel<T, 8, MOST, false>;
            launch_early(pass == kSquares ? squares_kernel<T, MOST> : pass == kMasters ? masters_kernel<T, MOST> : step,
                         (unsigned)(whole_chunks ? count : count * (t.chunk / kShort)), kThreads, 0, st, a);
        }
        first += n;
        at += count;
    }
}

void launch_pass(const ffcvb_adamw_args &a, const Tensors &t, Pass pass, cudaStream_t st) {
    with_type(a.type, [&](auto zero) {
        using T = decltype(zero);
        if (a.n_tensors <= 64)
            launch_all<T, 64>(a, t, pass, st);
        else
            launch_all<T, 1024>(a, t, pass, st);
    });
}

} // namespace

} // namespace ffcvb

using namespace ffcvb;

extern "C" {

int64_t ffcvb_adamw_layout(int32_t n, const int64_t *numel, int64_t *start, int64_t *sizes) {
    const long long chunk = chunk_size(n, numel);
    int64_t at = 0, chunks = 0;
    for (int32_t i = 0; i < n; i++) {
        start[i] = at;
        at += (numel[i] + kUnit - 1) / kUnit * kUnit;
        chunks += chunks_of(numel[i], chunk);
    }
    sizes[0] = n * (int64_t)sizeof(Tensor) + chunks * (int64_t)sizeof(Chunk);
    sizes[1] = chunks * (int64_t)sizeof(float);
    return at;
}

int ffcvb_adamw_table(int32_t n, const int64_t *numel, const uint64_t *params, void *table) {
    if (n < 0 || (n > 0 && (!numel || !params || !table))) return training_fail(FFCVB_E_ARG, "ffcvb_adamw_table: bad argument");
    Tensor *tensors = static_cast<Tensor *>(table);
    Chunk *to = reinterpret_cast<Chunk *>(tensors + n);
    const long long chunk = chunk_size(n, numel);
    int64_t at = 0;
    for (int32_t i = 0; i < n; i++) {
        if (chunks_of(numel[i], chunk) > 0x7fffffff) return training_fail(FFCVB_E_LIMIT, "ffcvb_adamw_table: tensor %d is too large", i);
        tensors[i] = Tensor{params[i], numel[i], at};
        at += (numel[i] + kUnit - 1) / kUnit * kUnit;
        for (int64_t c = 0; c < chunks_of(numel[i], chunk); c++) *to++ = Chunk{i, (int32_t)c};
    }
    return FFCVB_OK;
}

int ffcvb_adamw_step(const ffcvb_adamw_args *args, const int64_t *numel, int64_t *steps, const int32_t *group_of,
                     const uint64_t *grads, const ffcvb_adamw_group *groups, int32_t n_groups, void *stream) {
    if (!args || args->n_tensors < 0) return training_fail(FFCVB_E_ARG, "ffcvb_adamw_step: no arguments");
    const ffcvb_adamw_args &a = *args;
    if (a.n_tensors == 0) return FFCVB_OK;
    if (!numel || !grads || !steps || !group_of || !groups || !a.tensors || !a.exp_avg || !a.exp_avg_sq || (a.bits != 8 && a.bits != 32) ||
        (a.bits == 8 && !a.scales) || (a.type != FFCVB_TYPE_F32 && (!a.master || (a.type != FFCVB_TYPE_F16 && a.type != FFCVB_TYPE_BF16))) ||
        (a.max_norm > 0.0 && (!a.norm || !a.workspace)))
        return training_fail(FFCVB_E_ARG, "ffcvb_adamw_step: bad argument");
    Tensors t{numel, grads, steps, group_of, groups, 0, 0, chunk_size(a.n_tensors, numel)};
    for (int32_t i = 0; i < a.n_tensors; i++) {
        if (group_of[i] < 0 || group_of[i] >= n_groups) return training_fail(FFCVB_E_ARG, "ffcvb_adamw_step: tensor %d is in no group", i);
        t.values += numel[i];
        t.chunks += chunks_of(numel[i], t.chunk);
    }
    if (t.chunks * (t.chunk / kShort) > 0x7fffffff) return training_fail(FFCVB_E_LIMIT, "ffcvb_adamw_step: too many values");
    OnDevice here(a.device);
    if (!here.ok()) return training_fail(FFCVB_E_NODEVICE, "ffcvb_adamw_step: no device %d", a.device);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(st, &capture) != cudaSuccess) return launched("ffcvb_adamw_step");
    if (capture != cudaStreamCaptureStatusNone)
        return training_fail(FFCVB_E_ARG, "ffcvb_adamw_step: a step cannot be captured: its number, rates and gradients' addresses are its kernels' arguments");
    for (int32_t i = 0; i < a.n_tensors; i++) steps[i] += grads[i] != 0;
    if (a.max_norm > 0.0) {
        launch_pass(a, t, kSquares, st);
        launch_early(norm_kernel, 1, 1024, 0, st, static_cast<const float *>(a.workspace), t.chunks, a.norm);
    }
    launch_pass(a, t, kStep, st);
    return launched("ffcvb_adamw_step");
}

int ffcvb_adamw_masters(const ffcvb_adamw_args *args, const int64_t *numel, const uint64_t *which, void *stream) {
    if (!args || args->n_tensors < 0) return training_fail(FFCVB_E_ARG, "ffcvb_adamw_masters: no arguments");
    const ffcvb_adamw_args &a = *args;
    if (a.n_tensors == 0) return FFCVB_OK;
    if (!numel || !which || !a.tensors || !a.master || (a.type != FFCVB_TYPE_F16 && a.type != FFCVB_TYPE_BF16))
        return training_fail(FFCVB_E_ARG, "ffcvb_adamw_masters: bad argument");
    Tensors t{numel, which, nullptr, nullptr, nullptr, 0, 0, chunk_size(a.n_tensors, numel)};
    for (int32_t i = 0; i < a.n_tensors; i++) t.chunks += chunks_of(numel[i], t.chunk);
    if (t.chunks > 0x7fffffff) return training_fail(FFCVB_E_LIMIT, "ffcvb_adamw_masters: too many values");
    OnDevice here(a.device);
    if (!here.ok()) return training_fail(FFCVB_E_NODEVICE, "ffcvb_adamw_masters: no device %d", a.device);
    launch_pass(a, t, kMasters, static_cast<cudaStream_t>(stream));
    return launched("ffcvb_adamw_masters");
}

} // extern "C"
