// Rotary positions of queries and keys (sm_100a): pair (a, b) of a head at angle t becomes
// amplitude * (a cos t - b sin t, a sin t + b cos t).
// A CTA takes a tile of tokens: first the sines and cosines of all their pairs, once for all heads, into shared
// memory, then the heads.  Angles are counted in turns: the product of position and turns per position is made in 64 bits and
// whole turns are taken off there, which leaves nothing of a long context's angles to lose in 32.
#include "training.h"

namespace ffcvb {

namespace {

using Args = ffcvb_rotary_args;

constexpr int kThreads = 256;
constexpr int kTileAngles = 2048; // angles of a tile (16 KB)

template <typename T, int N, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads)
rotary_kernel(const __grid_constant__ Args a, int tile) {
    extern __shared__ float2 s_turn[]; // [tile][pairs]
    const int pairs = (int)(a.rotary_dim / 2);
    const long long tiles = (a.tokens + tile - 1) / tile;
    const long long b = blockIdx.x / tiles, first = blockIdx.x % tiles * tile;
    const int tokens = (int)min((long long)tile, a.tokens - first);
    for (int k = threadIdx.x; k < tokens * pairs; k += kThreads) {
        const int t = k / pairs, i = k % pairs;
        const long long at = b * a.positions_stride + (first + t) * a.axes + (a.axes == 2 && i >= pairs / 2);
        const double where = a.positions_float ? (double)static_cast<const float *>(a.positions)[at]
                                               : (double)static_cast<const int64_t *>(a.positions)[at];
        const double turns = where * a.turns[i];
        float sine, cosine;
        sincospif((float)(2.0 * (turns - rint(turns))), &sine, &cosine);
        s_turn[k] = make_float2(cosine * a.amplitude, (a.transpose ? -sine : sine) * a.amplitude);
    }
    __syncthreads();
    // slots of a head: packs (and their partners, half the rotated part on) that turn, then packs that are copied
    const int half = (int)a.rotary_dim / 2;
    const int turning = (INTERLEAVED ? (int)a.rotary_dim : half) / (INTERLEAVED && N == 1 ? 2 : N);
    const int slots = turning + (int)(a.head_dim - a.rotary_dim) / N;
    const int heads = (int)(a.heads + a.kv_heads);
    for (int k = threadIdx.x; k < tokens * heads * slots; k += kThreads) {
        const int slot = k % slots, h = k / slots % heads, t = k / slots / heads;
        const bool key = h >= a.heads;
        const int64_t *in_stride = key ? a.k_stride : a.q_stride, *out_stride = key ? a.k_out_stride : a.q_out_stride;
        const long long hh = key ? h - a.heads : h;
        const T *in = static_cast<const T *>(key ? a.k : a.q) + b * in_stride[0] + (first + t) * in_stride[1] + hh * in_stride[2];
        T *out = static_cast<T *>(key ? a.k_out : a.q_out) + b * out_stride[0] + (first + t) * out_stride[1] + hh * out_stride[2];
        const float2 *turn = s_turn + t * pairs;
        if (slot >= turning) {
            const int at = (int)a.rotary_dim + (slot - turning) * N;
            if (in != out) {
                Pack<T, N> p;
                p.load(in + at);
                p.store(out + at);
            }
        } else if (!INTERLEAVED || N == 1) {
            const int at = INTERLEAVED ? 2 * slot : slot * N, other = INTERLEAVED ? at + 1 : at + half;
            Pack<T, N> p, q;
            p.load(in + at);
            q.load(in + other);
            float u[N], v[N];
            p.get(u);
            q.get(v);
#pragma unroll
            for (int j = 0; j < N; j++) {
                const float2 cs = turn[slot * N + j];
                const float x = u[j] * cs.x - v[j] * cs.y;
                v[j] = u[j] * cs.y + v[j] * cs.x;
                u[j] = x;
            }
            p.set(u);
            q.set(v);
            p.store(out + at);
            q.store(out + other);
        } else {
            Pack<T, N> p;
            p.load(in + slot * N);
            float u[N];
            p.get(u);
#pragma unroll
            for (int j = 0; j + 1 < N; j += 2) {
                const float2 cs = turn[slot * (N / 2) + j / 2];
                const float x = u[j] * cs.x - u[j + 1] * cs.y;
                u[j + 1] = u[j] * cs.y + u[j + 1] * cs.x;
                u[j] = x;
            }
            p.set(u);
            p.store(out + slot * N);
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
    if (!a.positions || !a.turns || (a.heads > 0 && (!a.q || !a.q_out)) || (a.kv_heads > 0 && (!a.k || !a.k_out)))
        return training_fail(FFCVB_E_ARG, "ffcvb_rotary: bad argument");
    OnDevice here(a.device);
    if (!here.ok()) return training_fail(FFCVB_E_NODEVICE, "ffcvb_rotary: no device %d", a.device);
    const int pairs = (int)a.rotary_dim / 2;
    int tile = kTileAngles / pairs;
    if (tile > 16) tile = 16;
    if (tile < 1) tile = 1;
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
        const bool wide = (low & 15) == 0 && sizes % W == 0;
        auto run = [&](auto kernel) {
            kernel<<<(unsigned)ctas, kThreads, (size_t)tile * pairs * sizeof(float2), static_cast<cudaStream_t>(stream)>>>(a, tile);
        };
        if (wide)
            run(a.interleaved ? rotary_kernel<T, W, true> : rotary_kernel<T, W, false>);
        else
            run(a.interleaved ? rotary_kernel<T, 1, true> : rotary_kernel<T, 1, false>);
    });
    return launched("ffcvb_rotary");
}
