// Forward pass of the seam between two blocks (sm_100a): see norm_residual.cu.
#include "norm_residual.h"

namespace ffcvb {

namespace norms {

namespace {

// Two rows per CTA (or cluster, or warp) at a time, so that the sums of both take one barrier; with packs of 16 bytes those of the next
// rounds are on their way meanwhile.  POST: with an inner norm.
template <typename T, int N, bool MULTI, bool POST, int FORM>
__global__ void __launch_bounds__(MULTI ? 512 : 32, MULTI ? 1 : 16)
forward_kernel(const __grid_constant__ Args a, const Shape shape) {
    constexpr bool RING = N > 1;
    __shared__ __align__(16) float2 s_sum[72];
    extern __shared__ uint4 s_ring[]; // [ahead][2][streams][8 / N][threads]
    int rank = 0, cluster = blockIdx.x;
    if (MULTI && shape.ctas_per_row > 1) {
        rank = blockIdx.x % shape.ctas_per_row;
        cluster = blockIdx.x / shape.ctas_per_row;
    }
    const bool branch = FORM != kAny || a.h, normed = FORM != kAny || a.norm != FFCVB_NORM_NONE;
    const bool gated = FORM == kGated || (FORM == kAny && a.gate_kind != FFCVB_GATE_NONE);
    const bool per_sample = FORM == kGated || (FORM == kAny && a.gate_kind == FFCVB_GATE_SAMPLE);
    RowSum<MULTI> sum{s_sum, shape.ctas_per_row};
    sum.begin();
    wait_for_previous();
    const Columns<N, MULTI> c(a.width, shape.ctas_per_row, rank);
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
    const uint32_t mine = (uint32_t)__cvta_generic_to_shared(s_ring + threadIdx.x), slot_size = 2 * shape.streams * (8 / N) * blockDim.x * 16;
    const uint32_t ring_end = mine + shape.ahead * slot_size;
    const T *next_x = static_cast<const T *>(a.x) + begin * a.x_stride, *next_h = static_cast<const T *>(a.h) + begin * a.h_stride;
    auto fetch = [&](long long row, uint32_t to) {
#pragma unroll
        for (int i = 0; i < 2; i++)
            if (row + i < a.rows) {
                copy_packs(to, next_x + i * a.x_stride, c);
                if (branch) copy_packs(to, next_h + i * a.h_stride, c);
                if (gated) copy_packs(to, static_cast<const T *>(a.gate) + gate_row(row, i) * a.gate_stride, c);
            }
        copies_made();
        next_x += step * a.x_stride;
        next_h += step * a.h_stride;
        fetched();
    };
    if constexpr (RING)
        for (int k = 0; k < shape.ahead; k++) fetch(begin + k * step, mine + k * slot_size);
    let_next_begin();
    uint32_t slot = mine;
    T *to_y = static_cast<T *>(a.y) + begin * a.width, *to_z = static_cast<T *>(a.z) + begin * a.width;
    for (long long row = begin; row < a.rows; row += step, to_y += step * a.width, to_z += step * a.width) {
        const bool both = row + 1 < a.rows; // (else the second is whatever it is, and is not stored)
        Eight y[2], u[2], g[2];
        float4 stats[2] = {};
        if constexpr (RING) {
            copies_wait(shape.ahead);
            uint32_t from = slot;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                copied<T, N>(y[i], from);
                if (branch) copied<T, N>(u[i], from);
                if (gated) copied<T, N>(g[i], from);
            }
            fetch(row + shape.ahead * step, slot);
            slot += slot_size;
            if (slot == ring_end) slot = mine;
        } else {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int k = both ? i : 0;
                load_row<T>(y[i], a.x, (row + k) * a.x_stride, c);
                if (branch) load_row<T>(u[i], a.h, (row + k) * a.h_stride, c);
                if (gated) load_row<T>(g[i], a.gate, gate_row(row, k) * a.gate_stride, c);
            }
            fetched();
        }
        if (branch) {
            if (POST) {
                float mean[2], r[2];
                two_stats<N, MULTI>(u, a.post_norm, c, a.eps, sum, mean, r);
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
            two_stats<N, MULTI>(y, a.norm, c, a.eps, sum, mean, r);
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
    if (shape.threads == 32 && shape.ctas_per_row == 1)
        launch(forward_kernel<T, N, false, POST, FORM>, shape, room, stream, a, shape);
    else
        launch(forward_kernel<T, N, true, POST, FORM>, shape, room, stream, a, shape);
}

} // namespace

void launch_forward(const Args &a, const Shape &shape, bool wide, cudaStream_t stream) {
    const bool post = a.post_norm != FFCVB_NORM_NONE;
    const size_t room = wide ? (size_t)shape.threads * shape.ahead * 2 * shape.streams * 8 * type_size(a.type) : 0;
    with_type(a.type, [&](auto zero) {
        using T = decltype(zero);
        constexpr int W = 16 / (int)sizeof(T);
        auto formed = [&](auto post_norm) {
            constexpr bool P = decltype(post_norm)::value;
            if (!wide)
                sized<T, 1, P, kAny>(a, shape, room, stream);
            else if (form_of(a, false) == kPlain)
                sized<T, W, P, kPlain>(a, shape, room, stream);
            else if (form_of(a, false) == kGated)
                sized<T, W, P, kGated>(a, shape, room, stream);
            else
                sized<T, W, P, kAny>(a, shape, room, stream);
        };
        if (post)
            formed(Int<1>{});
        else
            formed(Int<0>{});
    });
}

} // namespace norms

} // namespace ffcvb
