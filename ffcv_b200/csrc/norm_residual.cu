// The seam between two blocks of a residual network, forward and backward (sm_100a):
//   u = post(h);  y = x + f u, f = number * scale * gate;  z = norm(y)
// A CTA holds one row in registers at a time, a thread the same columns of every row, so that weights are fetched once
// and the column sums of the backward pass stay in registers until the CTA's rows are through.  Backward, with
//   t = dy + r (g - mean g - yn mean(g yn)),  g = dz * weight, yn = (y - mean) r   (rms: without mean g)
// dx = t, the branch's gradient is du = t f, and the inner norm takes du on to dh by the same formula.  y is made
// again from x and h, in 32 bits: its rounded copy would cost the weights' gradients their last digits.
// Sums over columns of the gradient go through one partial row per CTA, added up in a fixed order by a second kernel.
//
// Reading and writing bounds it where rows are whole packs: 50432 bf16 rows of 768 with norm, branch and scale take 137 us
// forward and backward (118 at the rate of a copy), 8 of them for the columns' sums.  With an inner norm and gates
// (147520 rows of 1024) 532 us (461), where arithmetic and barriers between a row's sums show.
#include "norm_residual.h"

namespace ffcvb {

namespace norms {

namespace {

// Adds up partial rows: 32 columns per CTA, 32 rows at a time side by side (of 576 rows of 1024 columns 6 us; with 8 columns and 128 rows
// 9).  blockIdx.z: a run of the rows, whose sum goes to a partial row of its own.
struct Sums {
    const float *from[kColumns];
    void *to[kColumns];
    long long width, count, stride, run, to_z; // rows to add, from one to the next; rows of a run, and from one run's sum to the next one's
    int type;
};
__global__ void __launch_bounds__(1024)
add_up_kernel(const __grid_constant__ Sums s) {
    __shared__ float s_part[32][33];
    wait_for_previous();
    let_next_begin();
    const int lane = threadIdx.x & 31, beside = threadIdx.x >> 5;
    const long long c = blockIdx.x * 32ll + lane;
    const float *from = s.from[blockIdx.y];
    const long long begin = blockIdx.z * s.run, end = begin + s.run < s.count ? begin + s.run : s.count;
    float v = 0.0f;
    if (c < s.width) {
#pragma unroll 8
        for (long long r = begin + beside; r < end; r += 32) v += from[r * s.stride + c];
    }
    s_part[beside][lane] = v;
    __syncthreads();
    v = warp_sum(s_part[lane][beside]); // column `beside`
    const long long mine = blockIdx.x * 32ll + beside;
    if (lane == 0 && mine < s.width) {
        const long long at = blockIdx.z * s.to_z + mine;
        if (s.type == FFCVB_TYPE_F32)
            static_cast<float *>(s.to[blockIdx.y])[at] = v;
        else if (s.type == FFCVB_TYPE_F16)
            static_cast<__half *>(s.to[blockIdx.y])[at] = __float2half_rn(v);
        else
            static_cast<__nv_bfloat16 *>(s.to[blockIdx.y])[at] = __float2bfloat16_rn(v);
    }
}

// A gate's gradient per sample: the sums of its splits.
template <typename T>
__global__ void __launch_bounds__(256)
gates_kernel(const float *__restrict__ partial, T *__restrict__ dgate, long long width, long long splits, long long values) {
    wait_for_previous();
    const long long at = blockIdx.x * 256ll + threadIdx.x;
    if (at >= values) return;
    const long long sample = at / width;
    const float *from = partial + sample * splits * width + at % width;
    float v = 0.0f;
#pragma unroll 4
    for (long long k = 0; k < splits; k++) v += from[k * width];
    dgate[at] = from_float<T>(v);
}

bool wide_rows(const Args &a) {
    const int n = 16 / type_size(a.type);
    uintptr_t low = 0;
    for (const void *p : {a.x, a.h, a.gate, (const void *)a.y, (const void *)a.z, a.dy, a.dz, (const void *)a.dx, (const void *)a.dh, (const void *)a.dgate,
                          a.weight, a.bias, a.post_weight, a.post_bias, a.scale})
        low |= reinterpret_cast<uintptr_t>(p);
    return (low & 15) == 0 && (a.width | a.x_stride | (a.h ? a.h_stride : 0) | (a.gate ? a.gate_stride : 0) | (a.dy ? a.dy_stride : 0) |
                               (a.dz ? a.dz_stride : 0)) % n == 0;
}

// Rows of up to 4096 values are a CTA's (of up to 256 a warp's, 128 and 64 a half's and a quarter's), wider ones a cluster's; as many
// rounds ahead, at most `most_ahead`, as shared memory has room for, which 16 warps per SM share; besides: bytes per thread.
constexpr size_t kRoom = 208 * 1024;
Shape shape_of(const Args &a, bool wide, int streams, int rows, int most_ahead, size_t besides) {
    Shape s{};
    s.ctas_per_row = (int)((a.width + 4095) / 4096);
    const int eights = (int)((a.width + 7) / 8);
    s.threads = ((eights + s.ctas_per_row - 1) / s.ctas_per_row + 31) / 32 * 32;
    s.lanes = eights > 16 ? 32 : eights <= 8 ? 8 : 16;
    s.rows_at_once = kSms * (512 / s.threads) / s.ctas_per_row * s.rows_per_cta();
    s.streams = streams;
    const int size = type_size(a.type);
    auto ring = [&](int ahead) { // of a CTA
        if (wide) return (size_t)s.threads * ahead * rows * streams * 8 * size;
        const int threads = s.rows_per_cta() > 1 ? s.lanes : s.threads;
        return (size_t)(ahead + 1) * rows * streams * (size == 4 ? window_bytes<float>(threads) : window_bytes<__half>(threads)) * s.rows_per_cta();
    };
    for (s.ahead = most_ahead; s.ahead > 1 && 512 / s.threads * (ring(s.ahead) + besides * s.threads) > kRoom;) s.ahead--;
    s.ring = ring(s.ahead);
    return s;
}
Deal deal_of(const Args &a) {
    Deal d{};
    int streams = 0;
    for (const void *p : {a.x, a.h, a.dy, a.dz, a.gate_kind == FFCVB_GATE_TOKEN ? a.gate : nullptr}) streams += p != nullptr;
    d.shape = shape_of(a, wide_rows(a), streams, 1, 3, (a.gate_kind == FFCVB_GATE_SAMPLE ? 96 : 0) + (a.post_norm != FFCVB_NORM_NONE ? 64 : 0));
    const long long most = d.shape.rows_at_once;
    d.samples = a.gate_kind == FFCVB_GATE_SAMPLE ? a.rows / a.tokens : 1;
    d.tokens = a.gate_kind == FFCVB_GATE_SAMPLE ? a.tokens : a.rows;
    if (d.samples < 1) d.samples = 1; // no rows
    // splits of a sample: those with which the longest turn of a cluster is shortest
    const long long least = d.samples >= most ? 1 : most / d.samples, upto = d.samples >= most ? 8 : least;
    long long best = 0;
    d.splits = 1;
    for (long long s = least; s <= upto; s++) {
        const long long splits = s < d.tokens ? s : d.tokens > 1 ? d.tokens : 1;
        const long long turn = (d.samples * splits + most - 1) / most * ((d.tokens + splits - 1) / splits);
        if (!best || turn < best) {
            best = turn;
            d.splits = splits;
        }
    }
    d.units = d.samples * d.splits;
    const int per = d.shape.rows_per_cta();
    if (d.units < most) d.shape.rows_at_once = (int)((d.units + per - 1) / per * per);
    for (const void *p : {a.dweight, a.dbias, a.dpost_weight, a.dpost_bias, a.dscale}) d.columns += p != nullptr;
    // narrow rows have many partial rows and few columns: two steps then, the first with a CTA for every SM (128000 rows of 64 forward and
    // backward 33 us, 47 in one step; 394 rows of 192 11 us, 10 in one)
    const long long across = (a.width + 31) / 32 * d.columns, most_runs = across ? kSms / across : 0;
    d.runs = most_runs >= 4 && d.shape.rows_at_once >= 1024 ? (int)(most_runs < d.shape.rows_at_once / 128 ? most_runs : d.shape.rows_at_once / 128) : 1;
    return d;
}

int check(const Args *args, bool backward, const void *workspace) {
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
    if (backward && ((a.rows > 0 && !a.stats) || !workspace)) return training_fail(FFCVB_E_ARG, "%s: no statistics or workspace", name);
    if ((reinterpret_cast<uintptr_t>(a.stats) & 15) != 0) return training_fail(FFCVB_E_ARG, "%s: stats begin on 16 bytes", name);
    return FFCVB_OK;
}

} // namespace

} // namespace norms

} // namespace ffcvb

using namespace ffcvb;
using namespace ffcvb::norms;

extern "C" {

int ffcvb_norm_residual(const ffcvb_norm_residual_args *args, void *stream) {
    if (const int rc = check(args, false, nullptr)) return rc;
    const Args &a = *args;
    if (a.rows == 0) return FFCVB_OK;
    OnDevice here(a.device);
    if (!here.ok()) return training_fail(FFCVB_E_NODEVICE, "ffcvb_norm_residual: no device %d", a.device);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    Shape shape = shape_of(a, wide_rows(a), 1 + (a.h != nullptr) + (a.gate_kind != FFCVB_GATE_NONE), 2, 2, 0);
    const long long pairs = (a.rows + 1) / 2;
    const int per = shape.rows_per_cta();
    if (pairs < shape.rows_at_once) shape.rows_at_once = (int)((pairs + per - 1) / per * per);
    launch_forward(a, shape, wide_rows(a), st);
    return launched("ffcvb_norm_residual");
}

int64_t ffcvb_norm_residual_workspace(const ffcvb_norm_residual_args *args) {
    if (!args || args->rows < 0 || args->width < 1 || args->width > FFCVB_NORM_MAX_WIDTH || (args->gate_kind == FFCVB_GATE_SAMPLE && args->tokens < 1)) return 0;
    const Deal d = deal_of(*args);
    return (((int64_t)d.shape.rows_at_once + d.runs) * d.columns + (args->gate_kind == FFCVB_GATE_SAMPLE && d.splits > 1 ? d.units : 0)) * args->width * 4 + 16;
}

int ffcvb_norm_residual_backward(const ffcvb_norm_residual_args *args, void *workspace, void *stream) {
    if (const int rc = check(args, true, workspace)) return rc;
    const Args &a = *args;
    OnDevice here(a.device);
    if (!here.ok()) return training_fail(FFCVB_E_NODEVICE, "ffcvb_norm_residual_backward: no device %d", a.device);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const Deal d = deal_of(a);
    float *const room = static_cast<float *>(workspace);
    const long long row = d.columns * a.width;
    Partials part{room, room + d.shape.rows_at_once * row, room + (d.shape.rows_at_once + d.runs) * row};
    if (a.rows > 0) launch_backward(a, d, part, wide_rows(a), st);
    if (d.columns) {
        Sums s{};
        int n = 0;
        const bool twice = d.runs > 1 && a.rows > 0;
        for (void *p : {a.dweight, a.dbias, a.dpost_weight, a.dpost_bias, a.dscale})
            if (p) {
                s.from[n] = part.columns + n * a.width;
                s.to[n] = twice ? part.runs + n * a.width : p;
                n++;
            }
        s.width = a.width;
        s.count = a.rows > 0 ? d.shape.rows_at_once : 0;
        s.stride = s.to_z = row;
        s.run = twice ? (s.count + d.runs - 1) / d.runs : s.count;
        s.type = twice ? FFCVB_TYPE_F32 : a.param_type;
        const unsigned across = (unsigned)((a.width + 31) / 32);
        launch_early(add_up_kernel, dim3(across, n, twice ? d.runs : 1), 1024, 0, st, s);
        if (twice) {
            n = 0;
            for (void *p : {a.dweight, a.dbias, a.dpost_weight, a.dpost_bias, a.dscale})
                if (p) {
                    s.from[n] = part.runs + n * a.width;
                    s.to[n++] = p;
                }
            s.count = s.run = d.runs;
            s.type = a.param_type;
            launch_early(add_up_kernel, dim3(across, n), 1024, 0, st, s);
        }
    }
    if (a.dgate && a.gate_kind == FFCVB_GATE_SAMPLE && d.splits > 1 && a.rows > 0) // (then there are fewer samples than CTAs, or few splits)
        with_type(a.type, [&](auto zero) {
            using T = decltype(zero);
            const long long values = d.samples * a.width;
            launch_early(gates_kernel<T>, (unsigned)((values + 255) / 256), 256, 0, st, part.gate, static_cast<T *>(a.dgate), a.width, d.splits, values);
        });
    return launched("ffcvb_norm_residual_backward");
}

} // extern "C"
