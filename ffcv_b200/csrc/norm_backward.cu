// Backward pass of the seam between two blocks (sm_100a): see norm_residual.cu.
#include "norm_residual.h"

namespace ffcvb {

namespace norms {

namespace {

// One row per CTA (or cluster, or warp) at a time; with packs of 16 bytes those of the next are on their way meanwhile.
// POST: with an inner norm.  Of the branch's side two sums are kept per column and unit, A = sum t u and B = sum t (t with the gate,
// if it is one per token), u without weight and bias: all other gradients are made of them at a unit's end,
//   gate: f (pw A + pb B);  times the sample's gate:  scale: pw A + pb B,  post_weight: f A,  post_bias: f B.
template <typename T, int N, int LANES, bool POST, int FORM>
__global__ void __launch_bounds__(LANES ? 32 : 512, LANES ? 16 : 1)
backward_kernel(const __grid_constant__ Args a, const Deal deal, const Partials part) {
    constexpr bool PACKS = N > 1, MULTI = LANES == 0;
    const Shape &shape = deal.shape;
    __shared__ __align__(16) float2 s_sum[72];
    // [ahead][streams][8 / N][threads], or windows [rows][ahead + 1][streams]; with an inner norm its parameters, float4 [4][threads]; with
    // a gate per sample sums, floats [24][threads]
    extern __shared__ uint4 s_ring[];
    int rank;
    const int cluster = first_row<LANES>(shape, rank);
    RowSum<LANES> sum{s_sum, shape.ctas_per_row};
    sum.begin();
    wait_for_previous();
    const Columns<N, LANES> c(a.width, rank);
    const float over = 1.0f / (float)a.width;
    const bool per_sample = FORM == kGated || (FORM == kAny && a.gate_kind == FFCVB_GATE_SAMPLE);
    const bool per_token = FORM == kToken || (FORM == kAny && a.gate_kind == FFCVB_GATE_TOKEN);
    const bool branch = FORM != kAny || a.h, normed = FORM != kAny || a.norm != FFCVB_NORM_NONE;
    const bool given_dy = FORM != kAny || a.dy, given_dz = FORM != kAny || a.dz, want_dx = FORM != kAny || a.dx, want_dh = a.dh;
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(s_ring), window_size = window_bytes<T>(c.threads);
    const uint32_t slot_size = shape.streams * (PACKS ? (8 / N) * blockDim.x * 16 : window_size);
    const int slots = PACKS ? shape.ahead : shape.ahead + 1;
    const uint32_t mine = ring + (PACKS ? threadIdx.x * 16 : MULTI ? 0 : threadIdx.x / (MULTI ? 1 : LANES) * slots * slot_size), ring_end = mine + slots * slot_size;
    // with a gate per sample the sums over units are kept here, the thread's own
    float4 *const post = reinterpret_cast<float4 *>(s_ring + (PACKS ? shape.ahead * shape.streams * (8 / N) * blockDim.x : (int)(shape.ring / 16))) + threadIdx.x;
    float *const kept = reinterpret_cast<float *>(post - threadIdx.x + (POST ? 4 * blockDim.x : 0)) + threadIdx.x;
    const bool post_bias = a.post_bias;
    if (POST) { // (there are no registers for them)
        Eight pw, pb;
        load_params(pw, a.post_weight, a.param_type, c, 1.0f, 1.0f);
        load_params(pb, a.post_bias, a.param_type, c, 0.0f, 0.0f);
#pragma unroll
        for (int p = 0; p < 2; p++) {
            post[p * blockDim.x] = make_float4(pw[2 * p].lo(), pw[2 * p].hi(), pw[2 * p + 1].lo(), pw[2 * p + 1].hi());
            post[(p + 2) * blockDim.x] = make_float4(pb[2 * p].lo(), pb[2 * p].hi(), pb[2 * p + 1].lo(), pb[2 * p + 1].hi());
        }
    }
    auto post_params = [&](Eight &v, int bias) {
#pragma unroll
        for (int p = 0; p < 2; p++) {
            const float4 w = post[(p + 2 * bias) * blockDim.x];
            v[2 * p] = Two(w.x, w.y);
            v[2 * p + 1] = Two(w.z, w.w);
        }
    };
    if (per_sample)
        for (int k = 0; k < 24; k++) kept[k * blockDim.x] = 0.0f;
    Eight dw, db, sa, sb, w, f; // f: with the sample's gate; 0 beyond the row, which keeps everything of the branch 0 there
    fill(dw, 0.0f);
    fill(db, 0.0f);
    fill(sa, 0.0f);
    fill(sb, 0.0f);
    load_params(w, a.weight, a.param_type, c, 1.0f, 0.0f);
    auto load_f = [&]() {
        load_params(f, a.scale, a.param_type, c, 1.0f, 0.0f);
#pragma unroll
        for (int p = 0; p < kPairs; p++) f[p] = mul_rn(f[p], Two(a.number, a.number));
    };
    load_f();
    for (long long unit = cluster; unit < deal.units; unit += shape.rows_at_once) {
        const long long sample = unit / deal.splits, split = unit % deal.splits;
        const long long begin = sample * deal.tokens + deal.tokens * split / deal.splits;
        const long long end = sample * deal.tokens + deal.tokens * (split + 1) / deal.splits;
        if (per_sample) {
            Eight gate;
            load_f();
            load_row<T>(gate, a.gate, sample * a.gate_stride, c);
#pragma unroll
            for (int p = 0; p < kPairs; p++) f[p] = mul_rn(f[p], gate[p]);
        }
        const T *next_x = static_cast<const T *>(a.x) + begin * a.x_stride, *next_h = static_cast<const T *>(a.h) + begin * a.h_stride;
        const T *next_dy = static_cast<const T *>(a.dy) + begin * a.dy_stride, *next_dz = static_cast<const T *>(a.dz) + begin * a.dz_stride;
        auto fetch = [&](long long row, uint32_t to) {
            if (row < end) {
                auto copy = [&](const T *from) {
                    if constexpr (PACKS) {
                        copy_packs(to, from, c);
                    } else {
                        copy_window(to, from, c);
                        to += window_size;
                    }
                };
                copy(next_x);
                if (branch) copy(next_h);
                if (given_dy) copy(next_dy);
                if (given_dz) copy(next_dz);
                if (per_token) copy(static_cast<const T *>(a.gate) + row * a.gate_stride);
            }
            copies_made();
            next_x += a.x_stride;
            next_h += a.h_stride;
            next_dy += a.dy_stride;
            next_dz += a.dz_stride;
        };
        if (!PACKS) row_barrier<LANES>(sum.mask()); // (the unit before is through)
        for (int k = 0; k < shape.ahead; k++) fetch(begin + k, mine + k * slot_size);
        float4 next = {};
        if (begin < end) next = reinterpret_cast<const float4 *>(a.stats)[begin];
        uint32_t slot = mine;
        T *to_dx = static_cast<T *>(a.dx) + begin * a.width, *to_dh = static_cast<T *>(a.dh) + begin * a.width;
        for (long long row = begin; row < end; row++, to_dx += a.width, to_dh += a.width) {
            Eight y, u, t, dz, gate;
            const float4 stats = next;
            if (row + 1 < end) next = reinterpret_cast<const float4 *>(a.stats)[row + 1];
            if (!branch) fill(u, 0.0f);
            if (!given_dy) fill(t, 0.0f);
            if (!given_dz) fill(dz, 0.0f);
            copies_wait(shape.ahead);
            uint32_t from = slot;
            if constexpr (PACKS) {
                copied<T, N>(y, from);
                if (branch) copied<T, N>(u, from);
                if (given_dy) copied<T, N>(t, from);
                if (given_dz) copied<T, N>(dz, from);
                if (per_token) copied<T, N>(gate, from);
                fetch(row + shape.ahead, slot);
                slot += slot_size;
                if (slot == ring_end) slot = mine;
            } else {
                row_barrier<LANES>(sum.mask()); // (all have the row, and none the one before any more, whose place is the next one's)
                fetch(row + shape.ahead, slot == mine ? ring_end - slot_size : slot - slot_size);
                auto read = [&](Eight &v, const void *rows, long long stride) {
                    window(v, from, static_cast<const T *>(rows) + row * stride, c);
                    from += window_size;
                };
                read(y, a.x, a.x_stride);
                if (branch) read(u, a.h, a.h_stride);
                if (given_dy) read(t, a.dy, a.dy_stride);
                if (given_dz) read(dz, a.dz, a.dz_stride);
                if (per_token) read(gate, a.gate, a.gate_stride);
                slot += slot_size;
                if (slot == ring_end) slot = mine;
            }
            Eight pw;
            if (POST) {
                normalise(u, stats.z, stats.w); // without weight and bias
                post_params(pw, 0);
            }
            auto whole = [&](Eight &v) {
#pragma unroll
                for (int p = 0; p < kPairs; p++) v[p] = POST ? mul_rn(u[p], pw[p]) : u[p];
                if (POST && post_bias) {
                    Eight pb;
                    post_params(pb, 1);
#pragma unroll
                    for (int p = 0; p < kPairs; p++) v[p] = add_rn(v[p], pb[p]);
                }
            };
            if (normed) {
                Eight full;
                whole(full);
#pragma unroll
                for (int p = 0; p < kPairs; p++) y[p] = fma_rn(per_token ? mul_rn(full[p], gate[p]) : full[p], f[p], y[p]);
                normalise(y, stats.x, stats.y);
                Two first(0.0f, 0.0f), second(0.0f, 0.0f);
#pragma unroll
                for (int p = 0; p < kPairs; p++) {
                    dw[p] = fma_rn(dz[p], y[p], dw[p]);
                    db[p] = add_rn(db[p], dz[p]);
                    dz[p] = mul_rn(dz[p], w[p]);
                    first = add_rn(first, dz[p]);
                    second = fma_rn(dz[p], y[p], second);
                }
                const float2 means = sum(first.lo() + first.hi(), second.lo() + second.hi());
                const float m = a.norm == FFCVB_NORM_LAYER ? means.x * over : 0.0f, my = means.y * over;
                const Two minus_m(-m, -m), minus_my(-my, -my), r(stats.y, stats.y);
#pragma unroll
                for (int p = 0; p < kPairs; p++) t[p] = fma_rn(fma_rn(y[p], minus_my, add_rn(dz[p], minus_m)), r, t[p]);
            }
            if (want_dx) store_row<T>(t, to_dx, 0, c);
            if (!branch) continue;
            if (per_token) {
                Eight full, dgate;
                whole(full);
#pragma unroll
                for (int p = 0; p < kPairs; p++) {
                    dgate[p] = mul_rn(mul_rn(t[p], full[p]), f[p]);
                    t[p] = mul_rn(t[p], gate[p]);
                }
                if (a.dgate) store_row<T>(dgate, a.dgate, row * a.width, c);
            }
            Two first(0.0f, 0.0f), second(0.0f, 0.0f);
#pragma unroll
            for (int p = 0; p < kPairs; p++) {
                sa[p] = fma_rn(t[p], u[p], sa[p]);
                if (POST) sb[p] = add_rn(sb[p], t[p]);
                t[p] = mul_rn(t[p], f[p]);
                if (POST) {
                    t[p] = mul_rn(t[p], pw[p]);
                    first = add_rn(first, t[p]);
                    second = fma_rn(t[p], u[p], second);
                }
            }
            if (POST) {
                const float2 means = sum(first.lo() + first.hi(), second.lo() + second.hi());
                const float m = a.post_norm == FFCVB_NORM_LAYER ? means.x * over : 0.0f, mu = means.y * over;
                const Two minus_m(-m, -m), minus_mu(-mu, -mu), r(stats.w, stats.w);
#pragma unroll
                for (int p = 0; p < kPairs; p++) t[p] = mul_rn(fma_rn(u[p], minus_mu, add_rn(t[p], minus_m)), r);
            }
            if (want_dh) store_row<T>(t, to_dh, 0, c);
        }
        if (per_sample) {
            Eight dg, gate, pw, pb;
            load_params(pw, a.post_weight, a.param_type, c, 1.0f, 1.0f);
            load_params(pb, a.post_bias, a.param_type, c, 0.0f, 0.0f);
            load_row<T>(gate, a.gate, sample * a.gate_stride, c);
            load_f();
#pragma unroll
            for (int p = 0; p < kPairs; p++) {
                const Two whole = fma_rn(pw[p], sa[p], mul_rn(pb[p], sb[p])), fg = mul_rn(f[p], gate[p]);
                const Two add[3] = {mul_rn(fg, sa[p]), mul_rn(fg, sb[p]), mul_rn(gate[p], whole)};
#pragma unroll
                for (int j = 0; j < 6; j++) kept[(p * 6 + j) * blockDim.x] += add[j >> 1].half(j & 1);
                dg[p] = mul_rn(f[p], whole);
                sa[p] = sb[p] = Two(0.0f, 0.0f);
            }
            if (a.dgate && deal.splits == 1)
                store_row<T>(dg, a.dgate, sample * a.width, c);
            else if (a.dgate)
                store_floats(dg, part.gate + unit * a.width, c);
        }
    }
    let_next_begin();
    float *to = part.columns + (long long)cluster * deal.columns * a.width;
    auto put = [&](const Eight &v, const void *wanted) {
        if (!wanted) return;
        store_floats(v, to, c);
        to += a.width;
    };
    put(dw, a.dweight);
    put(db, a.dbias);
    Eight pw, pb;
    load_params(pw, a.post_weight, a.param_type, c, 1.0f, 1.0f);
    load_params(pb, a.post_bias, a.param_type, c, 0.0f, 0.0f);
#pragma unroll
    for (int p = 0; p < kPairs; p++) {
        const float *from = kept + p * 6 * blockDim.x;
        const int next = blockDim.x;
        if (per_sample) {
            dw[p] = Two(from[0], from[next]);
            db[p] = Two(from[2 * next], from[3 * next]);
            f[p] = Two(from[4 * next], from[5 * next]);
        } else {
            dw[p] = mul_rn(f[p], sa[p]);
            db[p] = mul_rn(f[p], sb[p]);
            f[p] = fma_rn(pw[p], sa[p], mul_rn(pb[p], sb[p]));
        }
        f[p] = mul_rn(f[p], Two(a.number, a.number));
    }
    put(dw, a.dpost_weight);
    put(db, a.dpost_bias);
    put(f, a.dscale);
}

template <typename T, int N, bool POST, int FORM>
void sized(const Args &a, const Deal &d, const Partials &part, size_t room, cudaStream_t stream) {
    auto run = [&](auto kernel) { launch(kernel, d.shape, room, stream, a, d, part); };
    if (d.shape.threads > 32 || d.shape.ctas_per_row > 1)
        run(backward_kernel<T, N, 0, POST, FORM>);
    else if (d.shape.lanes == 32)
        run(backward_kernel<T, N, 32, POST, FORM>);
    else if (d.shape.lanes == 16)
        run(backward_kernel<T, N, 16, POST, FORM>);
    else
        run(backward_kernel<T, N, 8, POST, FORM>);
}

} // namespace

void launch_backward(const Args &a, const Deal &d, const Partials &part, bool wide, cudaStream_t stream) {
    const bool post = a.post_norm != FFCVB_NORM_NONE;
    const size_t room = d.shape.ring + (size_t)d.shape.threads * ((post ? 64 : 0) + (a.gate_kind == FFCVB_GATE_SAMPLE ? 96 : 0));
    with_type(a.type, [&](auto zero) {
        using T = decltype(zero);
        with_form<T>(wide, post, form_of(a, true), [&](auto n, auto p, auto f) {
            sized<T, decltype(n)::value, (bool)decltype(p)::value, decltype(f)::value>(a, d, part, room, stream);
        });
    });
}

} // namespace norms

} // namespace ffcvb
