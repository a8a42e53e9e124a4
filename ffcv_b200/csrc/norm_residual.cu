// The seam between two blocks of a residual network, forward and backward (sm_100a):
//   u = post(h);  y = x + f u, f = number * scale * gate;  z = norm(y)
// A CTA holds one row in registers at a time, a thread the same columns of every row, so that weights are fetched once
// and the column sums of the backward pass stay in registers until the CTA's rows are through.  Backward, with
//   t = dy + r (g - mean g - yn mean(g yn)),  g = dz * weight, yn = (y - mean) r   (rms: without mean g)
// dx = t, the branch's gradient is du = t f, and the inner norm takes du on to dh by the same formula.  y is made
// again from x and h, in 32 bits: its rounded copy would cost the weights' gradients their last digits.
// Sums over columns of the gradient go through one partial row per CTA, added up in a fixed order by a second kernel.
#include "training.h"

namespace ffcvb {

namespace {

using Args = ffcvb_norm_residual_args;

template <int N>
__device__ __forceinline__ void load_params(float (&v)[N], const void *p, int type, long long at, long long width, float otherwise) {
#pragma unroll
    for (int j = 0; j < N; j++) {
        v[j] = otherwise;
        if (p && at + j < width) {
            if (type == FFCVB_TYPE_F32)
                v[j] = static_cast<const float *>(p)[at + j];
            else if (type == FFCVB_TYPE_F16)
                v[j] = to_float(static_cast<const __half *>(p)[at + j]);
            else
                v[j] = to_float(static_cast<const __nv_bfloat16 *>(p)[at + j]);
        }
    }
}

// Sums over a row's threads; every second call may use the other half of `s`, so that one barrier is enough.
struct RowSum {
    float *s; // [2][2][32]
    int turn = 0;
    __device__ __forceinline__ float2 operator()(float a, float b) {
        a = warp_sum(a);
        b = warp_sum(b);
        const int warps = blockDim.x >> 5;
        if (warps == 1) return make_float2(a, b);
        float *to = s + turn * 64;
        turn ^= 1;
        if ((threadIdx.x & 31) == 0) {
            to[threadIdx.x >> 5] = a;
            to[32 + (threadIdx.x >> 5)] = b;
        }
        __syncthreads();
        const int lane = threadIdx.x & 31;
        return make_float2(warp_sum(lane < warps ? to[lane] : 0.0f), warp_sum(lane < warps ? to[32 + lane] : 0.0f));
    }
};

// Mean (0 for rms) and 1 / deviation of a row: the mean first, then the squares of what is left.
template <int N, int VPT>
__device__ __forceinline__ float2 row_stats(const float (&v)[VPT][N], int kind, long long width, float eps, RowSum &sum) {
    float mean = 0.0f;
    if (kind == FFCVB_NORM_LAYER) {
        float a = 0.0f;
#pragma unroll
        for (int k = 0; k < VPT; k++)
#pragma unroll
            for (int j = 0; j < N; j++) a += v[k][j];
        mean = sum(a, 0.0f).x / (float)width;
    }
    float q = 0.0f;
#pragma unroll
    for (int k = 0; k < VPT; k++) {
        const long long at = ((long long)k * blockDim.x + threadIdx.x) * N;
#pragma unroll
        for (int j = 0; j < N; j++)
            if (at + j < width) q += (v[k][j] - mean) * (v[k][j] - mean);
    }
    return make_float2(mean, 1.0f / sqrtf(sum(q, 0.0f).x / (float)width + eps));
}

template <typename T, int N, int VPT>
__device__ __forceinline__ void load_row(float (&v)[VPT][N], const void *p, long long offset, long long width) {
#pragma unroll
    for (int k = 0; k < VPT; k++) {
        const long long at = ((long long)k * blockDim.x + threadIdx.x) * N;
        if (p && at < width) {
            Pack<T, N> pack;
            pack.load(static_cast<const T *>(p) + offset + at);
            pack.get(v[k]);
        } else {
#pragma unroll
            for (int j = 0; j < N; j++) v[k][j] = 0.0f;
        }
    }
}
template <typename T, int N, int VPT>
__device__ __forceinline__ void store_row(const float (&v)[VPT][N], void *p, long long offset, long long width) {
#pragma unroll
    for (int k = 0; k < VPT; k++) {
        const long long at = ((long long)k * blockDim.x + threadIdx.x) * N;
        if (at < width) {
            Pack<T, N> pack;
            pack.set(v[k]);
            pack.store(static_cast<T *>(p) + offset + at);
        }
    }
}

// WIDE loads (N > 1) need rows of a multiple of N values on 16-byte boundaries.
template <typename T, int N, int VPT>
__global__ void __launch_bounds__(1024, 1)
forward_kernel(const __grid_constant__ Args a) {
    __shared__ float s_sum[128];
    RowSum sum{s_sum};
    float w[VPT][N], b[VPT][N], pw[VPT][N], pb[VPT][N], f[VPT][N];
#pragma unroll
    for (int k = 0; k < VPT; k++) {
        const long long at = ((long long)k * blockDim.x + threadIdx.x) * N;
        load_params<N>(w[k], a.weight, a.param_type, at, a.width, 1.0f);
        load_params<N>(b[k], a.bias, a.param_type, at, a.width, 0.0f);
        load_params<N>(pw[k], a.post_weight, a.param_type, at, a.width, 1.0f);
        load_params<N>(pb[k], a.post_bias, a.param_type, at, a.width, 0.0f);
        load_params<N>(f[k], a.scale, a.param_type, at, a.width, 1.0f);
    }
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        float y[VPT][N];
        float4 stats = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        load_row<T, N, VPT>(y, a.x, row * a.x_stride, a.width);
        if (a.h) {
            float u[VPT][N], gate[VPT][N];
            load_row<T, N, VPT>(u, a.h, row * a.h_stride, a.width);
            if (a.gate_kind != FFCVB_GATE_NONE)
                load_row<T, N, VPT>(gate, a.gate, (a.gate_kind == FFCVB_GATE_SAMPLE ? row / a.tokens : row) * a.gate_stride, a.width);
            if (a.post_norm != FFCVB_NORM_NONE) {
                const float2 inner = row_stats<N, VPT>(u, a.post_norm, a.width, a.eps, sum);
                stats.z = inner.x;
                stats.w = inner.y;
#pragma unroll
                for (int k = 0; k < VPT; k++)
#pragma unroll
                    for (int j = 0; j < N; j++) u[k][j] = (u[k][j] - inner.x) * inner.y * pw[k][j] + pb[k][j];
            }
#pragma unroll
            for (int k = 0; k < VPT; k++)
#pragma unroll
                for (int j = 0; j < N; j++)
                    y[k][j] += u[k][j] * (a.number * f[k][j] * (a.gate_kind != FFCVB_GATE_NONE ? gate[k][j] : 1.0f));
            if (a.y) store_row<T, N, VPT>(y, a.y, row * a.width, a.width);
        }
        if (a.norm != FFCVB_NORM_NONE) {
            // (columns beyond the row hold 0 times nothing: x is 0 there and so is u times its factor, except for a bias)
#pragma unroll
            for (int k = 0; k < VPT; k++) {
                const long long at = ((long long)k * blockDim.x + threadIdx.x) * N;
#pragma unroll
                for (int j = 0; j < N; j++)
                    if (at + j >= a.width) y[k][j] = 0.0f;
            }
            const float2 outer = row_stats<N, VPT>(y, a.norm, a.width, a.eps, sum);
            stats.x = outer.x;
            stats.y = outer.y;
#pragma unroll
            for (int k = 0; k < VPT; k++)
#pragma unroll
                for (int j = 0; j < N; j++) y[k][j] = (y[k][j] - outer.x) * outer.y * w[k][j] + b[k][j];
            store_row<T, N, VPT>(y, a.z, row * a.width, a.width);
        }
        if (a.stats && threadIdx.x == 0) reinterpret_cast<float4 *>(a.stats)[row] = stats;
    }
}

// How the backward pass deals its rows out.  A unit is a run of rows of one sample (with a gate per sample, whose
// gradient is a sum over them) or of all rows.
struct Deal {
    long long samples, tokens, splits, units;
    int ctas, columns; // column sums of each CTA: weight, bias, post_weight, post_bias, scale
};
// Partial rows: [ctas][columns][width] of the column sums, then [units][width] of the gate's with more than one split.
struct Partials {
    float *columns, *gate;
};

constexpr int kColumns = 5;

template <typename T, int N, int VPT, int MAX_THREADS>
__global__ void __launch_bounds__(MAX_THREADS, 1)
backward_kernel(const __grid_constant__ Args a, const Deal deal, const Partials part) {
    __shared__ float s_sum[128];
    RowSum sum{s_sum};
    float w[VPT][N], pw[VPT][N], pb[VPT][N], f[VPT][N];
    float dw[VPT][N] = {}, db[VPT][N] = {}, dpw[VPT][N] = {}, dpb[VPT][N] = {}, df[VPT][N] = {};
#pragma unroll
    for (int k = 0; k < VPT; k++) {
        const long long at = ((long long)k * blockDim.x + threadIdx.x) * N;
        load_params<N>(w[k], a.weight, a.param_type, at, a.width, 1.0f);
        load_params<N>(pw[k], a.post_weight, a.param_type, at, a.width, 1.0f);
        load_params<N>(pb[k], a.post_bias, a.param_type, at, a.width, 0.0f);
        load_params<N>(f[k], a.scale, a.param_type, at, a.width, 1.0f);
    }
    const float over = 1.0f / (float)a.width;
    const bool gated = a.gate_kind != FFCVB_GATE_NONE;
    for (long long unit = blockIdx.x; unit < deal.units; unit += gridDim.x) {
        const long long sample = unit / deal.splits, split = unit % deal.splits;
        const long long begin = sample * deal.tokens + deal.tokens * split / deal.splits;
        const long long end = sample * deal.tokens + deal.tokens * (split + 1) / deal.splits;
        float gate[VPT][N], dg[VPT][N] = {};
        if (a.gate_kind == FFCVB_GATE_SAMPLE) load_row<T, N, VPT>(gate, a.gate, sample * a.gate_stride, a.width);
        for (long long row = begin; row < end; row++) {
            float y[VPT][N], u[VPT][N], t[VPT][N], dz[VPT][N];
            load_row<T, N, VPT>(y, a.x, row * a.x_stride, a.width);
            load_row<T, N, VPT>(u, a.h, row * a.h_stride, a.width);
            load_row<T, N, VPT>(t, a.dy, row * a.dy_stride, a.width);
            load_row<T, N, VPT>(dz, a.dz, row * a.dz_stride, a.width);
            if (a.gate_kind == FFCVB_GATE_TOKEN) load_row<T, N, VPT>(gate, a.gate, row * a.gate_stride, a.width);
            const float4 stats = reinterpret_cast<const float4 *>(a.stats)[row];
            if (a.post_norm != FFCVB_NORM_NONE) // u: normalised, without weight and bias
#pragma unroll
                for (int k = 0; k < VPT; k++)
#pragma unroll
                    for (int j = 0; j < N; j++) u[k][j] = (u[k][j] - stats.z) * stats.w;
            if (a.norm != FFCVB_NORM_NONE) {
                float mean_g = 0.0f, mean_gy = 0.0f;
#pragma unroll
                for (int k = 0; k < VPT; k++)
#pragma unroll
                    for (int j = 0; j < N; j++) {
                        const float factor = a.number * f[k][j] * (gated ? gate[k][j] : 1.0f);
                        y[k][j] = (y[k][j] + (u[k][j] * pw[k][j] + pb[k][j]) * factor - stats.x) * stats.y;
                        mean_g += dz[k][j] * w[k][j];
                        mean_gy += dz[k][j] * w[k][j] * y[k][j];
                        dw[k][j] += dz[k][j] * y[k][j];
                        db[k][j] += dz[k][j];
                    }
                const float2 means = sum(mean_g, mean_gy);
                const float m = a.norm == FFCVB_NORM_LAYER ? means.x * over : 0.0f, my = means.y * over;
#pragma unroll
                for (int k = 0; k < VPT; k++) {
                    const bool in = ((long long)k * blockDim.x + threadIdx.x) * N < a.width; // (a pack is in or not)
#pragma unroll
                    for (int j = 0; j < N; j++) t[k][j] = in ? t[k][j] + stats.y * (dz[k][j] * w[k][j] - m - y[k][j] * my) : 0.0f;
                }
            }
            if (a.dx) store_row<T, N, VPT>(t, a.dx, row * a.width, a.width);
            if (!a.h) continue;
            float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
            for (int k = 0; k < VPT; k++)
#pragma unroll
                for (int j = 0; j < N; j++) {
                    const float whole = u[k][j] * pw[k][j] + pb[k][j], g = gated ? gate[k][j] : 1.0f;
                    const float tu = a.number * t[k][j] * whole;
                    df[k][j] += tu * g;
                    if (a.gate_kind == FFCVB_GATE_SAMPLE) dg[k][j] += tu * f[k][j];
                    if (a.gate_kind == FFCVB_GATE_TOKEN) dz[k][j] = tu * f[k][j]; // (dz is not needed any more)
                    t[k][j] *= a.number * f[k][j] * g;
                    dpw[k][j] += t[k][j] * u[k][j];
                    dpb[k][j] += t[k][j];
                    s1 += t[k][j] * pw[k][j];
                    s2 += t[k][j] * pw[k][j] * u[k][j];
                }
            if (a.gate_kind == FFCVB_GATE_TOKEN && a.dgate) store_row<T, N, VPT>(dz, a.dgate, row * a.width, a.width);
            if (a.post_norm != FFCVB_NORM_NONE) {
                const float2 means = sum(s1, s2);
                const float m = a.post_norm == FFCVB_NORM_LAYER ? means.x * over : 0.0f, mu = means.y * over;
#pragma unroll
                for (int k = 0; k < VPT; k++)
#pragma unroll
                    for (int j = 0; j < N; j++) t[k][j] = stats.w * (t[k][j] * pw[k][j] - m - u[k][j] * mu);
            }
            if (a.dh) store_row<T, N, VPT>(t, a.dh, row * a.width, a.width);
        }
        if (a.gate_kind == FFCVB_GATE_SAMPLE && a.dgate) {
            if (deal.splits == 1) {
                store_row<T, N, VPT>(dg, a.dgate, sample * a.width, a.width);
            } else {
#pragma unroll
                for (int k = 0; k < VPT; k++) {
                    const long long at = ((long long)k * blockDim.x + threadIdx.x) * N;
#pragma unroll
                    for (int j = 0; j < N; j++)
                        if (at + j < a.width) part.gate[unit * a.width + at + j] = dg[k][j];
                }
            }
        }
    }
    void *const wanted[kColumns] = {a.dweight, a.dbias, a.dpost_weight, a.dpost_bias, a.dscale};
    float *to = part.columns + (long long)blockIdx.x * deal.columns * a.width;
#pragma unroll
    for (int c = 0; c < kColumns; c++) {
        if (!wanted[c]) continue;
#pragma unroll
        for (int k = 0; k < VPT; k++) {
            const long long at = ((long long)k * blockDim.x + threadIdx.x) * N;
            const float(&v)[N] = c == 0 ? dw[k] : c == 1 ? db[k] : c == 2 ? dpw[k] : c == 3 ? dpb[k] : df[k];
#pragma unroll
            for (int j = 0; j < N; j++)
                if (at + j < a.width) to[at + j] = v[j];
        }
        to += a.width;
    }
}

// Adds up partial rows: 32 columns per CTA, eight runs of rows side by side.
struct Sums {
    const float *from[kColumns];
    void *to[kColumns];
    long long width, count, stride, from_z, to_z; // rows to add, from one to the next; from one sum (blockIdx.z) to the next
    int type;
};
__global__ void __launch_bounds__(256)
add_up_kernel(const __grid_constant__ Sums s) {
    __shared__ float s_part[8][33];
    const int lane = threadIdx.x & 31, run = threadIdx.x >> 5;
    const long long c = blockIdx.x * 32ll + lane;
    const float *from = s.from[blockIdx.y] + blockIdx.z * s.from_z;
    float v = 0.0f;
    if (c < s.width)
        for (long long r = run; r < s.count; r += 8) v += from[r * s.stride + c];
    s_part[run][lane] = v;
    __syncthreads();
    if (run == 0 && c < s.width) {
#pragma unroll
        for (int k = 1; k < 8; k++) v += s_part[k][lane];
        const long long at = blockIdx.z * s.to_z + c;
        if (s.type == FFCVB_TYPE_F32)
            static_cast<float *>(s.to[blockIdx.y])[at] = v;
        else if (s.type == FFCVB_TYPE_F16)
            static_cast<__half *>(s.to[blockIdx.y])[at] = __float2half_rn(v);
        else
            static_cast<__nv_bfloat16 *>(s.to[blockIdx.y])[at] = __float2bfloat16_rn(v);
    }
}

bool wide_rows(const Args &a) {
    const int n = 16 / type_size(a.type);
    uintptr_t low = 0;
    for (const void *p : {a.x, a.h, a.gate, (const void *)a.y, (const void *)a.z, a.dy, a.dz, (const void *)a.dx, (const void *)a.dh, (const void *)a.dgate})
        low |= reinterpret_cast<uintptr_t>(p);
    return (low & 15) == 0 && (a.width | a.x_stride | (a.h ? a.h_stride : 0) | (a.gate ? a.gate_stride : 0) | (a.dy ? a.dy_stride : 0) |
                               (a.dz ? a.dz_stride : 0)) % n == 0;
}

// Packs of a row per thread, so that a row has at most 1024 threads.
int packs_per_thread(long long packs) {
    int per = 1;
    while (packs > 1024ll * per) per *= 2;
    return per;
}
int threads_of(long long packs, int per) { return (int)((packs + per - 1) / per + 31) / 32 * 32; }

// CTAs that a backward pass is dealt out to: about 24 warps per SM.
Deal deal_of(const Args &a) {
    Deal d{};
    const long long packs = wide_rows(a) ? a.width / (16 / type_size(a.type)) : a.width;
    const int threads = threads_of(packs, packs_per_thread(packs));
    const long long most = (long long)kSms * (threads >= 768 ? 1 : 768 / threads);
    d.samples = a.gate_kind == FFCVB_GATE_SAMPLE ? a.rows / a.tokens : 1;
    d.tokens = a.gate_kind == FFCVB_GATE_SAMPLE ? a.tokens : a.rows;
    if (d.samples < 1) d.samples = 1; // no rows
    d.splits = d.samples >= most ? 1 : (most + d.samples - 1) / d.samples;
    if (d.splits > d.tokens) d.splits = d.tokens;
    if (d.splits < 1) d.splits = 1;
    d.units = d.samples * d.splits;
    d.ctas = (int)(d.units < most ? d.units : most);
    for (const void *p : {a.dweight, a.dbias, a.dpost_weight, a.dpost_bias, a.dscale}) d.columns += p != nullptr;
    return d;
}

int check(const Args *args, bool backward) {
    const char *name = backward ? "ffcvb_norm_residual_backward" : "ffcvb_norm_residual";
    if (!args) return training_fail(FFCVB_E_ARG, "%s: no arguments", name);
    const Args &a = *args;
    auto type_ok = [](int t) { return t == FFCVB_TYPE_F32 || t == FFCVB_TYPE_F16 || t == FFCVB_TYPE_BF16; };
    auto norm_ok = [](int n) { return n >= FFCVB_NORM_NONE && n <= FFCVB_NORM_RMS; };
    if (a.width > FFCVB_NORM_MAX_WIDTH) return training_fail(FFCVB_E_LIMIT, "%s: rows of more than %d values", name, FFCVB_NORM_MAX_WIDTH);
    if (a.rows < 0 || a.width < 1 || !type_ok(a.type) || !type_ok(a.param_type) || !norm_ok(a.norm) || !norm_ok(a.post_norm) ||
        a.gate_kind < FFCVB_GATE_NONE || a.gate_kind > FFCVB_GATE_TOKEN)
        return training_fail(FFCVB_E_ARG, "%s: bad size, type or kind", name);
    if (a.rows > 0 && (!a.x || (a.gate_kind != FFCVB_GATE_NONE && !a.gate) || (!a.h && (a.post_norm != FFCVB_NORM_NONE || a.gate_kind != FFCVB_GATE_NONE || a.scale)) ||
                       (!a.h && a.norm == FFCVB_NORM_NONE)))
        return training_fail(FFCVB_E_ARG, "%s: bad argument", name);
    if ((a.gate_kind == FFCVB_GATE_SAMPLE && (a.tokens < 1 || a.rows % a.tokens)))
        return training_fail(FFCVB_E_ARG, "%s: bad argument", name);
    if (!backward && a.rows > 0 && ((a.norm != FFCVB_NORM_NONE && !a.z) || (a.h && !a.y)))
        return training_fail(FFCVB_E_ARG, "%s: no room for the results", name);
    if (backward && ((a.rows > 0 && !a.stats) || !a.workspace)) return training_fail(FFCVB_E_ARG, "%s: no statistics or workspace", name);
    return FFCVB_OK;
}

} // namespace

} // namespace ffcvb

using namespace ffcvb;

extern "C" {

int ffcvb_norm_residual(const ffcvb_norm_residual_args *args, void *stream) {
    if (const int rc = check(args, false)) return rc;
    const Args &a = *args;
    if (a.rows == 0) return FFCVB_OK;
    OnDevice here(a.device);
    if (!here.ok()) return training_fail(FFCVB_E_NODEVICE, "ffcvb_norm_residual: no device %d", a.device);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    with_type(a.type, [&](auto zero) {
        using T = decltype(zero);
        constexpr int W = 16 / (int)sizeof(T);
        const bool wide = wide_rows(a);
        const long long packs = wide ? a.width / W : a.width;
        const int per = packs_per_thread(packs), threads = threads_of(packs, per);
        const long long most = (long long)kSms * (2048 / threads < 32 ? 2048 / threads : 32);
        auto run = [&](auto kernel) { kernel<<<(unsigned)(a.rows < most ? a.rows : most), threads, 0, st>>>(a); };
        if (wide)
            run(per == 1 ? forward_kernel<T, W, 1> : per == 2 ? forward_kernel<T, W, 2> : forward_kernel<T, W, 4>);
        else
            run(per == 1 ? forward_kernel<T, 1, 1> : per <= 4 ? forward_kernel<T, 1, 4> : forward_kernel<T, 1, 16>);
    });
    return launched("ffcvb_norm_residual");
}

int64_t ffcvb_norm_residual_workspace(const ffcvb_norm_residual_args *args) {
    if (!args || args->rows < 0 || args->width < 1 || (args->gate_kind == FFCVB_GATE_SAMPLE && args->tokens < 1)) return 0;
    const Deal d = deal_of(*args);
    return ((int64_t)d.ctas * d.columns + (args->gate_kind == FFCVB_GATE_SAMPLE && d.splits > 1 ? d.units : 0)) * args->width * 4 + 16;
}

int ffcvb_norm_residual_backward(const ffcvb_norm_residual_args *args, void *stream) {
    if (const int rc = check(args, true)) return rc;
    const Args &a = *args;
    OnDevice here(a.device);
    if (!here.ok()) return training_fail(FFCVB_E_NODEVICE, "ffcvb_norm_residual_backward: no device %d", a.device);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const Deal d = deal_of(a);
    Partials part{static_cast<float *>(a.workspace), static_cast<float *>(a.workspace) + (long long)d.ctas * d.columns * a.width};
    if (a.rows > 0)
        with_type(a.type, [&](auto zero) {
            using T = decltype(zero);
            constexpr int W = 16 / (int)sizeof(T);
            const bool wide = wide_rows(a);
            const long long packs = wide ? a.width / W : a.width;
            const int per = packs_per_thread(packs), threads = threads_of(packs, per);
            auto run = [&](auto kernel) { kernel<<<d.ctas, threads, 0, st>>>(a, d, part); };
            if (wide && per == 1)
                run(threads <= 256 ? backward_kernel<T, W, 1, 256> : backward_kernel<T, W, 1, 1024>);
            else if (wide)
                run(per == 2 ? backward_kernel<T, W, 2, 1024> : backward_kernel<T, W, 4, 1024>);
            else
                run(per == 1 ? backward_kernel<T, 1, 1, 1024> : per <= 4 ? backward_kernel<T, 1, 4, 1024> : backward_kernel<T, 1, 16, 1024>);
        });
    Sums s{};
    int n = 0;
    for (void *p : {a.dweight, a.dbias, a.dpost_weight, a.dpost_bias, a.dscale})
        if (p) {
            s.from[n] = part.columns + n * a.width;
            s.to[n++] = p;
        }
    s.width = a.width;
    s.count = a.rows > 0 ? d.ctas : 0;
    s.stride = d.columns * a.width;
    s.type = a.param_type;
    const unsigned across = (unsigned)((a.width + 31) / 32);
    if (n) add_up_kernel<<<dim3(across, n), 256, 0, st>>>(s);
    if (a.dgate && a.gate_kind == FFCVB_GATE_SAMPLE && d.splits > 1 && a.rows > 0) {
        Sums g{};
        g.from[0] = part.gate;
        g.to[0] = a.dgate;
        g.width = g.stride = g.to_z = a.width;
        g.count = d.splits;
        g.from_z = d.splits * a.width;
        g.type = a.type;
        // (more than one split means that there are fewer samples than CTAs)
        add_up_kernel<<<dim3(across, 1, (unsigned)d.samples), 256, 0, st>>>(g);
    }
    return launched("ffcvb_norm_residual_backward");
}

} // extern "C"
