// Rotary positions of queries and keys (sm_100a): pair (a, b) of a head at angle t becomes
// amplitude * (a cos t - b sin t, a sin t + b cos t).
// A CTA takes a tile of tokens: first the sines and cosines of all their pairs, once for all heads, into shared
// memory, then the heads.  Angles are counted in turns.  Whole positions multiply turns in units of 2^-64 of a turn: the product's low
// 64 bits are what is left of it without whole turns, whatever the position.  Positions that are floats multiply in 64-bit floats.  The
// nearest quarter turn is taken off before the rest is rounded to 24 bits, which is then 2^-28 of a turn off at most.  (Root of the mean square of a turned value's error in 32 bits, positions 0 to 65535: 3.9e-8, 5.6e-8 with the whole
// angle rounded; 3.7e-8 with sines and cosines that are rounded once.)
//
// Reading and writing bounds it: 65536 tokens of 40 half-turned bf16 heads of 128 take 231 us each way, 205 at the rate of a copy; with
// the tile's rows asked into the L2 while the angles are made 278.
#include "training.h"
#include "two.h"

namespace ffcvb {

namespace {

using Args = ffcvb_rotary_args;

constexpr int kThreads = 256;
constexpr int kTileAngles = 4096; // angles of a tile at most (32 KB)
constexpr int kTileBytes = 32 * 1024; // of queries and keys of a tile at least, where that many angles allow it

// (a, b) -> (a c - b s, a s + b c) for pairs of either.
__device__ __forceinline__ void turn(Two &a, Two &b, Two c, Two s) {
    const Two x = fma_rn(b, s, mul_rn(a, c)); // (s: with the sign of the first)
    b = fma_rn(a, mul_rn(s, Two(-1.0f, -1.0f)), mul_rn(b, c));
    a = x;
}

// A head's slots: packs that turn (with their partners, half the rotated part on), then packs that are copied.  A thread has the same slot of the same
// head of several tokens, one after the other; where a token has fewer slots than a CTA threads, tokens lie side by side.
template <typename T, int N, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads, 5)
rotary_kernel(const __grid_constant__ Args a, int tile) {
    // tokens that a thread has on their way: four packs (with eight 65536 tokens of 40 half-turned heads of 128 take 667 us, not 462)
    constexpr int kAtOnce = INTERLEAVED || N * sizeof(T) < 16 ? 4 : 2;
    extern __shared__ float s_cos[]; // [tile][pairs], then the sines
    wait_for_previous();
    let_next_begin();
    const int pairs = (int)a.rotary_dim / 2;
    float *const s_sin = s_cos + tile * pairs;
    const long long tiles = (a.tokens + tile - 1) / tile;
    const long long b = blockIdx.x / tiles, first = blockIdx.x % tiles * tile;
    const int tokens = (int)min((long long)tile, a.tokens - first);
    // a thread makes the angles of one pair, of several tokens, or (more pairs than threads) of several pairs
    const int across = min(pairs, kThreads), beside = kThreads / across;
    for (int i = threadIdx.x % across; i < pairs && threadIdx.x < across * beside; i += across) {
        const double turns = a.turns[i];
        const uint64_t steps = a.steps[i];
        const long long begin = b * a.positions_stride + first * a.axes + (a.axes == 2 && i >= pairs / 2);
#pragma unroll 2
        for (int t = threadIdx.x / across; t < tokens; t += beside) {
            const long long at = begin + t * a.axes;
            float angle; // what the nearest quarter turn leaves, in half turns, -1/4 .. 1/4
            int quarters;
            if (a.positions_float) {
                const double turned = static_cast<const float *>(a.positions)[at] * turns, four = 4.0 * (turned - rint(turned)), whole = rint(four);
                angle = (float)(0.5 * (four - whole));
                quarters = (int)whole;
            } else {
                const uint64_t turned = (uint64_t)static_cast<const int64_t *>(a.positions)[at] * steps;
                quarters = (int)((turned + (1ull << 61)) >> 62);
                angle = (float)(int64_t)(turned - ((uint64_t)quarters << 62)) * 1.0842021724855044e-19f; // 2^-63
            }
            float sine, cosine;
            sincospif(angle, &sine, &cosine);
            if (quarters & 1) {
                const float was = sine;
                sine = cosine;
                cosine = -was;
            }
            if (quarters & 2) {
                sine = -sine;
                cosine = -cosine;
            }
            s_cos[t * pairs + i] = cosine * a.amplitude;
            s_sin[t * pairs + i] = (a.transpose ? sine : -sine) * a.amplitude;
        }
    }
    __syncthreads();
    constexpr int PER = INTERLEAVED && N == 1 ? 2 : N; // values of a turning slot, or of a half of it
    const int half = (int)a.rotary_dim / 2;
    const int turning = (INTERLEAVED ? (int)a.rotary_dim : half) / PER;
    const int slots = turning + (int)(a.head_dim - a.rotary_dim) / N;
    const int items = (int)(a.heads + a.kv_heads) * slots;
    const int abreast = items < kThreads ? kThreads / items : 1; // tokens side by side
    for (int item = items < kThreads ? threadIdx.x % items : threadIdx.x; item < items; item += kThreads) {
        int t = items < kThreads ? threadIdx.x / items : 0;
        if (t >= abreast) return;
        const int slot = item % slots, h = item / slots;
        const bool key = h >= a.heads;
        const int64_t *in_stride = key ? a.k_stride : a.q_stride, *out_stride = key ? a.k_out_stride : a.q_out_stride;
        const long long head = key ? h - a.heads : h;
        const bool turns = slot < turning;
        const int at = turns ? slot * PER : (int)a.rotary_dim + (slot - turning) * N;
        const int other = INTERLEAVED ? 1 : half; // from a value to its partner, where it is in another pack
        const T *in = static_cast<const T *>(key ? a.k : a.q) + b * in_stride[0] + (first + t) * in_stride[1] + head * in_stride[2] + at;
        T *out = static_cast<T *>(key ? a.k_out : a.q_out) + b * out_stride[0] + (first + t) * out_stride[1] + head * out_stride[2] + at;
        const long long in_step = abreast * in_stride[1], out_step = abreast * out_stride[1];
        if (!turns && in == out) continue;
        constexpr bool TWO = !INTERLEAVED || N == 1; // partners in two packs
        for (; t < tokens; t += kAtOnce * abreast, in += kAtOnce * in_step, out += kAtOnce * out_step) {
            Pack<T, N> p[kAtOnce], q[kAtOnce];
#pragma unroll
            for (int i = 0; i < kAtOnce; i++)
                if (t + i * abreast < tokens) {
                    p[i].load(in + i * in_step);
                    if (TWO && turns) q[i].load(in + i * in_step + other);
                }
#pragma unroll
            for (int i = 0; i < kAtOnce; i++) {
                if (t + i * abreast >= tokens) break;
                if (turns) {
                    const int angle = (t + i * abreast) * pairs + (INTERLEAVED ? slot * PER / 2 : slot * N);
                    const float *c = s_cos + angle, *s = s_sin + angle;
                    if constexpr (N == 1) {
                        float u[1], v[1];
                        p[i].get(u);
                        q[i].get(v);
                        const float x[1] = {u[0] * c[0] + v[0] * s[0]}, y[1] = {v[0] * c[0] - u[0] * s[0]};
                        p[i].set(x);
                        q[i].set(y);
                    } else if constexpr (INTERLEAVED) {
                        float u[N];
                        p[i].get(u);
#pragma unroll
                        for (int j = 0; j < N; j += 2) {
                            const Two x = fma_rn(Two(u[j + 1], u[j]), Two(s[j / 2], -s[j / 2]), mul_rn(Two(u[j], u[j + 1]), Two(c[j / 2], c[j / 2])));
                            u[j] = x.lo();
                            u[j + 1] = x.hi();
                        }
                        p[i].set(u);
                    } else {
                        float u[N], v[N];
                        p[i].get(u);
                        q[i].get(v);
                        if constexpr (N == 2) {
                            Two x(u[0], u[1]), y(v[0], v[1]);
                            turn(x, y, Two(c[0], c[1]), Two(s[0], s[1]));
                            u[0] = x.lo(), u[1] = x.hi(), v[0] = y.lo(), v[1] = y.hi();
                        }
#pragma unroll
                        for (int j = 0; j + 3 < N; j += 4) {
                            const float4 cc = *reinterpret_cast<const float4 *>(c + j), ss = *reinterpret_cast<const float4 *>(s + j);
                            Two u0(u[j], u[j + 1]), u1(u[j + 2], u[j + 3]), v0(v[j], v[j + 1]), v1(v[j + 2], v[j + 3]);
                            turn(u0, v0, Two(cc.x, cc.y), Two(ss.x, ss.y));
                            turn(u1, v1, Two(cc.z, cc.w), Two(ss.z, ss.w));
                            u[j] = u0.lo(), u[j + 1] = u0.hi(), u[j + 2] = u1.lo(), u[j + 3] = u1.hi();
                            v[j] = v0.lo(), v[j + 1] = v0.hi(), v[j + 2] = v1.lo(), v[j + 3] = v1.hi();
                        }
                        p[i].set(u);
                        q[i].set(v);
                    }
                }
                p[i].store(out + i * out_step);
                if (TWO && turns) q[i].store(out + i * out_step + other);
            }
        }
    }
}

} // namespace

} // namespace ffcvb

using namespace ffcvb;

extern "C" int ffcvb_rotary(const ffcvb_rotary_args *args, void *stream) {
    if (!args) return training_fail(FFCVB_E_ARG, "ffcvb_rotary: no arguments");
    const Args &a = *args;
    if (a.batch < 0 || a.tokens < 0 || a.heads < 0 || a.kv_heads < 0 || a.head_dim < 2 || a.head_dim > 4096 || a.rotary_dim < 2 || a.rotary_dim > a.head_dim ||
        (a.axes != 1 && a.axes != 2) || a.rotary_dim % (2 * a.axes) || a.heads + a.kv_heads > 0xffff || (a.type != FFCVB_TYPE_F32 && a.type != FFCVB_TYPE_F16 && a.type != FFCVB_TYPE_BF16))
        return training_fail(FFCVB_E_ARG, "ffcvb_rotary: bad size or type");
    if (a.batch * a.tokens * (a.heads + a.kv_heads) == 0) return FFCVB_OK;
    if (!a.positions || !a.turns || !a.steps || (a.heads > 0 && (!a.q || !a.q_out)) || (a.kv_heads > 0 && (!a.k || !a.k_out)))
        return training_fail(FFCVB_E_ARG, "ffcvb_rotary: bad argument");
    OnDevice here(a.device);
    if (!here.ok()) return training_fail(FFCVB_E_NODEVICE, "ffcvb_rotary: no device %d", a.device);
    const int pairs = (int)a.rotary_dim / 2;
    const long long token = (a.heads + a.kv_heads) * a.head_dim * type_size(a.type);
    int tile = (int)(kTileBytes / token);
    if (tile < 16) tile = 16;
    if (tile > kTileAngles / pairs) tile = kTileAngles / pairs;
    if (tile < 1) tile = 1;
    // fewer tokens per CTA where there are few: two CTAs for every SM
    while (tile > 2 && a.batch * ((a.tokens + tile - 1) / tile) < 2 * kSms) tile /= 2;
    const long long ctas = a.batch * ((a.tokens + tile - 1) / tile);
    if (ctas > 0x7fffffff) return training_fail(FFCVB_E_LIMIT, "ffcvb_rotary: too many tokens");
    with_type(a.type, [&](auto zero) {
        using T = decltype(zero);
        constexpr int W = 16 / (int)sizeof(T);
        uintptr_t low = 0;
        long long sizes = a.head_dim | a.rotary_dim | (a.interleaved ? 0 : a.rotary_dim / 2);
        for (int k = 0; k < 3; k++)
            sizes |= (a.heads ? a.q_stride[k] | a.q_out_stride[k] : 0) | (a.kv_heads ? a.k_stride[k] | a.k_out_stride[k] : 0);
        if (a.heads) low |= reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.q_out);
        if (a.kv_heads) low |= reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.k_out);
        const bool wide = (low & 15) == 0 && sizes % W == 0, half_wide = (low & 7) == 0 && sizes % (W / 2) == 0;
        auto run = [&](auto kernel) {
            launch_early(kernel, (unsigned)ctas, kThreads, (size_t)tile * pairs * 2 * sizeof(float), static_cast<cudaStream_t>(stream), a, tile);
        };
        if (wide)
            run(a.interleaved ? rotary_kernel<T, W, true> : rotary_kernel<T, W, false>);
        else if (half_wide)
            run(a.interleaved ? rotary_kernel<T, W / 2, true> : rotary_kernel<T, W / 2, false>);
        else
            run(a.interleaved ? rotary_kernel<T, 1, true> : rotary_kernel<T, 1, false>);
    });
    return launched("ffcvb_rotary");
}
