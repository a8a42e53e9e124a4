// Forward pass of the seam between two blocks (sm_100a): see norm_residual.cu.
#include "norm_residual.h"

namespace ffcvb {

namespace norms {

namespace {

// Two rows per CTA (or cluster, or warp) at a time, so that the sums of both take one barrier; with packs of 16 bytes those of the next
// rounds are on their way meanwhile.  POST: with an inner norm.
template <typename T, int N, int LANES, bool POST, int FORM>
__global__ void __launch_bounds__(LANES ? 32 : 512, LANES ? 16 : 1)
forward_kernel(const __grid_constant__ Args a, const Shape shape) {
    constexpr bool PACKS = N > 1, MULTI = LANES == 0;
    __shared__ __align__(16) float2 s_sum[72];
    extern __shared__ uint4 s_ring[]; // [ahead][2][streams][8 / N][threads], or windows [rows][ahead + 1][2][streams]
    int rank;
    const int cluster = first_row<LANES>(shape, rank);
    const bool branch = FORM != kAny || a.h, normed = FORM != kAny || a.norm != FFCVB_NORM_NONE;
    const bool gated = FORM == kGated || FORM == kToken || (FORM == kAny && a.gate_kind != FFCVB_GATE_NONE);
    const bool per_sample = FORM == kGated || (FORM == kAny && a.gate_kind == FFCVB_GATE_SAMPLE);
    RowSum<LANES> sum{s_sum, shape.ctas_per_row};
    sum.begin();
    wait_for_previous();
    const Columns<N, LANES> c(a.width, rank);
    Eight w, b, f, pw, pb; // (f is 0 beyond the row, which keeps y 0 there)
    load_params(w, a.weight, a.param_type, c, 1.0f, 1.0f);
    load_params(b, a.bias, a.param_type, c, 0.0f, 0.0f);
    load_params(f, a.scale, a.param_type, c, 1.0f, 0.0f);
    if (POST) {
        load_params(pw, a.post_weight, a.param_type, c, 1.0f, 1.0f);
        load_params(pb, a.post_bias, a.param_type, c, 0.0f, 0.0f);
    }
#pragma unroll
    for (int p = 0; p < kPairs; p++) f[p] = mul_rn(f[p], Two(a.number, a.number));
    const long long step = 2ll * shape.rows_at_once, begin = 2ll * cluster;
    // the sample of the next row to be fetched, and the row's place in it
    long long next_sample = per_sample ? begin / a.tokens : 0, next_place = per_sample ? begin % a.tokens : 0;
    const long long sample_step = per_sample ? step / a.tokens : 0, place_step = per_sample ? step % a.tokens : 0;
    auto gate_row = [&](long long row, int i) { return per_sample ? next_sample + (i && next_place + 1 == a.tokens) : row + i; };
    auto fetched = [&]() {
        if (!per_sample) return;
        next_sample += sample_step;
        next_place += place_step;
        if (next_place >= a.tokens) {
            next_place -= a.tokens;
            next_sample++;
        }
    };
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(s_ring), window_size = window_bytes<T>(c.threads);
    const uint32_t slot_size = 2 * shape.streams * (PACKS ? (8 / N) * blockDim.x * 16 : window_size);
    const int slots = PACKS ? shape.ahead : shape.ahead + 1;
    const uint32_t mine = ring + (PACKS ? threadIdx.x * 16 : MULTI ? 0 : threadIdx.x / (MULTI ? 1 : LANES) * slots * slot_size), ring_end = mine + slots * slot_size;
    const T *next_x = static_cast<const T *>(a.x) + begin * a.x_stride, *next_h = static_cast<const T *>(a.h) + begin * a.h_stride;
    auto fetch = [&](long long row, uint32_t to) {
#pragma unroll
        for (int i = 0; i < 2; i++)
            if (row + i < a.rows) {
                auto copy = [&](const T *from) {
                    if constexpr (PACKS) {
                        copy_packs(to, from, c);
                    } else {
                        copy_window(to, from, c);
                        to += window_size;
                    }
                };
                copy(next_x + i * a.x_stride);
                if (branch) copy(next_h + i * a.h_stride);
                if (gated) copy(static_cast<const T *>(a.gate) + gate_row(row, i) * a.gate_stride);
            }
        copies_made();
        next_x += step * a.x_stride;
        next_h += step * a.h_stride;
        fetched();
    };
    for (int k = 0; k < shape.ahead; k++) fetch(begin + k * step, mine + k * slot_size);
    long long sample = per_sample ? begin / a.tokens : 0, place = per_sample ? begin % a.tokens : 0; // of the row in hand (windows)
    let_next_begin();
    uint32_t slot = mine;
    T *to_y = static_cast<T *>(a.y) + begin * a.width, *to_z = static_cast<T *>(a.z) + begin * a.width;
    for (long long row = begin; row < a.rows; row += step, to_y += step * a.width, to_z += step * a.width) {
        const bool both = row + 1 < a.rows; // (else the second is whatever it is, and is not stored)
        Eight y[2], u[2], g[2];
        float4 stats[2] = {};
        copies_wait(shape.ahead);
        uint32_t from = slot;
        if constexpr (PACKS) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                copied<T, N>(y[i], from);
                if (branch) copied<T, N>(u[i], from);
                if (gated) copied<T, N>(g[i], from);
            }
            fetch(row + shape.ahead * step, slot);
        } else {
            row_barrier<LANES>(sum.mask()); // (all have the row, and none the one before any more, whose place is the next one's)
            fetch(row + shape.ahead * step, slot == mine ? ring_end - slot_size : slot - slot_size);
#pragma unroll
            for (int i = 0; i < 2; i++) {
                if (i == 1 && !both) break;
                auto read = [&](Eight &v, const void *rows, long long stride, long long which) {
                    window(v, from, static_cast<const T *>(rows) + which * stride, c);
                    from += window_size;
                };
                read(y[i], a.x, a.x_stride, row + i);
                if (branch) read(u[i], a.h, a.h_stride, row + i);
                if (gated) read(g[i], a.gate, a.gate_stride, per_sample ? sample + (i && place + 1 == a.tokens) : row + i);
            }
            if (!both) {
                fill(y[1], 0.0f);
                fill(u[1], 0.0f);
                fill(g[1], 0.0f);
            }
            if (per_sample) {
                sample += sample_step;
                place += place_step;
                if (place >= a.tokens) {
                    place -= a.tokens;
                    sample++;
                }
            }
        }
        slot += slot_size;
        if (slot == ring_end) slot = mine;
        if (branch) {
            if (POST) {
                float mean[2], r[2];
                two_stats<N, LANES>(u, a.post_norm, c, a.eps, sum, mean, r);
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    stats[i].z = mean[i];
                    stats[i].w = r[i];
                    normalise(u[i], mean[i], r[i]);
#pragma unroll
                    for (int p = 0; p < kPairs; p++) u[i][p] = fma_rn(u[i][p], pw[p], pb[p]);
                }
            }
#pragma unroll
            for (int i = 0; i < 2; i++) {
                if (gated)
#pragma unroll
                    for (int p = 0; p < kPairs; p++) u[i][p] = mul_rn(u[i][p], g[i][p]);
#pragma unroll
                for (int p = 0; p < kPairs; p++) y[i][p] = fma_rn(u[i][p], f[p], y[i][p]);
                if (i == 0 || both) store_row<T>(y[i], to_y, i * a.width, c);
            }
        }
        if (normed) {
            float mean[2], r[2];
            two_stats<N, LANES>(y, a.norm, c, a.eps, sum, mean, r);
#pragma unroll
            for (int i = 0; i < 2; i++) {
                stats[i].x = mean[i];
                stats[i].y = r[i];
                normalise(y[i], mean[i], r[i]);
#pragma unroll
                for (int p = 0; p < kPairs; p++) y[i][p] = fma_rn(y[i][p], w[p], b[p]);
                if (i == 0 || both) store_row<T>(y[i], to_z, i * a.width, c);
            }
        }
        if (c.first == 0) {
            reinterpret_cast<float4 *>(a.stats)[row] = stats[0];
            if (both) reinterpret_cast<float4 *>(a.stats)[row + 1] = stats[1];
        }
    }
}

template <typename T, int N, bool POST, int FORM>
void sized(const Args &a, const Shape &shape, size_t room, cudaStream_t stream) {
    auto run = [&](auto kernel) { launch(kernel, shape, room, stream, a, shape); };
    if (shape.threads > 32 || shape.ctas_per_row > 1)
        run(forward_kernel<T, N, 0, POST, FORM>);
    else if (shape.lanes == 32)
        run(forward_kernel<T, N, 32, POST, FORM>);
    else if (shape.lanes == 16)
        run(forward_kernel<T, N, 16, POST, FORM>);
    else
        run(forward_kernel<T, N, 8, POST, FORM>);
}

} // namespace

void launch_forward(const Args &a, const Shape &shape, bool wide, cudaStream_t stream) {
    const bool post = a.post_norm != FFCVB_NORM_NONE;
    const size_t room = shape.ring;
    with_type(a.type, [&](auto zero) {
        using T = decltype(zero);
        with_form<T>(wide, post, form_of(a, false), [&](auto n, auto p, auto f) {
            sized<T, decltype(n)::value, (bool)decltype(p)::value, decltype(f)::value>(a, shape, room, stream);
        });
    });
}

} // namespace norms

} // namespace ffcvb
