// Cross entropy of a linear layer's outputs, which are not kept, with the gradients of what goes in (sm_100a).
//
// With hidden values x [rows, width], weights w [classes, width] and a bias b the logits are z = x w^T + b, a row's loss is S lse(z) - sum T z
// (see cross_entropy.cu) and G = S exp(z - lse) - T the gradient of its logits; then dx = G w, dw = G^T x, db = sum of G's rows.  All are
// matrix products on the tensor cores with sums of 32 bits: x w^T a first time, whose tiles never leave the SM: of 128 logits of a row the
// largest and the sum of exponentials relative to it are left; joined, they give the loss and lse.  Then x w^T a second time, whose
// tiles leave as G, rounded to 16 bits (one rounding of at most 2^-9 (bf16) of a value that is multiplied and added with thousands of others), for as many
// classes at once as the workspace has room for; of these dx's part is added up and dw's rows are finished.  So 8 * rows * classes * width
// operations instead of 6 are done, and the logits, of any size, take a bounded workspace.
#include "losses.h"
#include "tensor.h"

#include <algorithm>

namespace ffcvb {

namespace {

constexpr int kThreads = 320; // a warp that copies, one that multiplies, eight that take the results
constexpr int kSum = 64;      // of the sum's terms in a stage: 128 bytes
constexpr uint32_t kRowsBytes = 128 * 128, kStagingBytes = 8 * 4096;
template <int BN> constexpr int kStages = BN == 256 ? 4 : 6;
template <int BN> constexpr uint32_t kStageBytes = kRowsBytes + BN * 128;
// stages, the eight warps' staging, the bias of a tile, barriers; and what it takes to begin on 1024 bytes
template <int BN> constexpr uint32_t kRoom = kStages<BN> * kStageBytes<BN> + kStagingBytes + 1024 + 256 + 1024;

enum { kStatistics, kGradient, kProducts };      // what a kernel makes of its products
enum { kWritten, kWritten32, kAdded32 };         // how products leave: as they are to be, or as parts in 32 bits
enum { kFixed, kRowsCounted, kSumCounted };      // what depends on the number of rows that count

// One product A B of matrices, in tiles of 128 by BN, the sum in `splits` parts.
struct alignas(64) Product {
    CUtensorMap a, b, c;
    int row_tiles, column_tiles, sum_blocks, splits;
    int a_along_sum; // A's rows in memory run along the sum
    int leaves, counted;
    int b_first;     // where B begins along the sum (kProducts), or its rows (else)
    int c_rows, c_last; // C's rows of a part; and of those there are
    int unused[6];
};

struct Head {
    ffcvb_linear_cross_entropy_args a;
    const int *map;      // rows that count, or NULL: all
    const int *place;    // a row's place among them, or -1
    const float *counted;
    float2 *parts;       // [classes / (BN / 2)][rows_pad]: largest logit and sum of exponentials
    float *parts_apart;  // the same: sum of logits relative to the largest; with smoothing
    float *bias_parts;   // [rows_pad / 32][chunk]
    const float *most;   // largest upstream of a row
    int rows_pad, first, columns; // classes of this chunk
    int part_count, part_columns;
};

struct Products {
    Product of[2];
    int count;
    int unused[15];
    Head head;
};

// G is held times this: in fp16 shares of less than 2^-24 of a row would be lost.
template <typename T> constexpr float kHeld = 1.0f;
template <> constexpr float kHeld<__half> = 32768.0f;

template <typename T> __device__ __forceinline__ uint32_t two_of(float lo, float hi);
template <> __device__ __forceinline__ uint32_t two_of<__half>(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
}
template <> __device__ __forceinline__ uint32_t two_of<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
}

__device__ __forceinline__ int rows_counted(const Head &h) { return h.counted ? (int)*h.counted : (int)h.a.rows; }

// What all gradients are multiplied by behind the sums.
template <typename T> __device__ __forceinline__ float gradient_scale(const Head &h) {
    float k = h.a.scale / kHeld<T>;
    if (h.a.upstream) k *= h.a.upstream_per_row ? *h.most : *h.a.upstream;
    if (h.a.mean) k /= h.counted ? fmaxf(*h.counted, 1.0f) : (float)h.a.rows;
    return k;
}

// A tile: of which product, where, and its part of the sum.
struct Tile {
    int product, row, column, from, to, split;
};
template <int MODE> __device__ __forceinline__ bool tile_at(const Products &p, long long t, int rows, Tile &tile) {
    for (int i = 0; i < (MODE == kProducts ? p.count : 1); i++) {
        const Product &w = p.of[i];
        const int row_tiles = w.counted == kRowsCounted ? (rows + 127) / 128 : w.row_tiles;
        const long long here = (long long)row_tiles * w.column_tiles * w.splits;
        if (t >= here) {
            t -= here;
            continue;
        }
        tile.product = i;
        if (MODE == kProducts) { // tiles of the same rows beside one another
            tile.column = (int)(t % w.column_tiles);
            t /= w.column_tiles;
            tile.row = (int)(t % row_tiles);
            tile.split = (int)(t / row_tiles);
        } else { // tiles of the same weights
            tile.row = (int)(t % row_tiles);
            tile.column = (int)(t / row_tiles);
            tile.split = 0;
        }
        const int blocks = w.counted == kSumCounted ? (rows + kSum - 1) / kSum : w.sum_blocks, each = (blocks + w.splits - 1) / w.splits;
        tile.from = min(tile.split * each, blocks);
        tile.to = min(tile.from + each, blocks);
        return true;
    }
    return false;
}

// A CTA per SM that takes tile after tile.  Products of the next tile go into the other half of TMEM while eight warps, two for each 32 rows, take
// the last one's.  A wait that does not end makes the CTA give up: all that it has not finished is NaN, and it ends.
template <int MODE, typename T, int BN>
__global__ void __launch_bounds__(kThreads, 1) products_kernel(const __grid_constant__ Products p) {
    constexpr int STAGES = kStages<BN>, HALF = BN / 2;
    extern __shared__ uint8_t s_room[];
    const uint32_t room = (shared_address(s_room) + 1023) & ~1023u, staging = room + STAGES * kStageBytes<BN>;
    float *s_bias = (float *)(s_room + (staging + kStagingBytes - shared_address(s_room)));
    volatile int *s_gave_up = (volatile int *)(s_bias + 256);
    const uint32_t s_tmem = shared_address(s_bias + 257), bars = shared_address(s_bias + 260);
    const uint32_t full = bars, empty = bars + 8 * STAGES, done = bars + 16 * STAGES, taken = done + 16, drained = taken + 16;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; s++) {
            barrier_init(full + 8 * s, 1);
            barrier_init(empty + 8 * s, 1);
        }
        for (int s = 0; s < 2; s++) {
            barrier_init(done + 8 * s, 1);
            barrier_init(taken + 8 * s, 8);
        }
        barrier_init(drained, 1);
        *s_gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc(s_tmem, 2 * BN);
    tmem_before_sync();
    __syncthreads();
    tmem_after_sync();
    wait_for_previous();
    let_next_begin();
    const Head &h = p.head;
    const uint32_t tmem = *(volatile uint32_t *)(s_bias + 257);
    const int rows = rows_counted(h);
    Tile tile;
    if (warp == 0) {
        if (lane == 0) {
            uint32_t n = 0; // stages filled so far
            bool fine = true;
            for (long long t = blockIdx.x; fine && tile_at<MODE>(p, t, rows, tile); t += gridDim.x) {
                const Product &w = p.of[tile.product];
                for (int k = tile.from; k < tile.to; k++, n++) {
                    const uint32_t s = n % STAGES, at = room + s * kStageBytes<BN>, bar = full + 8 * s;
                    fine = n < STAGES || barrier_wait(empty + 8 * s, (n / STAGES - 1) & 1, s_gave_up);
                    if (!fine) break;
                    barrier_expect(bar, kStageBytes<BN>);
                    if (MODE == kProducts) {
                        if (w.a_along_sum) {
                            copy_box(at, &w.a, tile.row * 128, k * kSum, bar);
                            copy_box(at + kRowsBytes / 2, &w.a, tile.row * 128 + 64, k * kSum, bar);
                        } else {
                            copy_box(at, &w.a, k * kSum, tile.row * 128, bar);
                        }
#pragma unroll
                        for (int j = 0; j < BN / 64; j++)
                            copy_box(at + kRowsBytes + j * (kSum * 128), &w.b, tile.column * BN + 64 * j, w.b_first + k * kSum, bar);
                    } else {
                        copy_box(at, &w.a, k * kSum, tile.row * 128, bar);
                        copy_box(at + kRowsBytes, &w.b, k * kSum, w.b_first + tile.column * BN, bar);
                    }
                }
            }
            if (!fine) // no copy arrives behind the CTA's end
                for (uint32_t k = n < STAGES ? 0 : n - STAGES; k < n; k++) {
                    volatile int patient = 0;
                    barrier_wait(full + 8 * (k % STAGES), k / STAGES & 1, &patient);
                }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (lane == 0) {
            uint32_t n = 0, m = 0; // stages and tiles multiplied so far
            bool fine = true;
            for (long long t = blockIdx.x; fine && tile_at<MODE>(p, t, rows, tile); t += gridDim.x) {
                if (tile.from >= tile.to) continue;
                const bool a_along_sum = MODE == kProducts && p.of[tile.product].a_along_sum;
                const uint32_t kind = product_kind(sizeof(T) == 2 && kHeld<T> == 1.0f, BN, a_along_sum, MODE == kProducts), half = m & 1;
                fine = m < 2 || barrier_wait(taken + 8 * half, (m / 2 - 1) & 1, s_gave_up);
                if (!fine) break;
                tmem_after_sync();
                for (int k = tile.from; k < tile.to; k++, n++) {
                    const uint32_t s = n % STAGES, at = room + s * kStageBytes<BN>;
                    fine = barrier_wait(full + 8 * s, n / STAGES & 1, s_gave_up);
                    if (!fine) break;
                    tmem_after_sync();
                    const uint64_t a = operand(at, kSum * 128), b = operand(at + kRowsBytes, kSum * 128);
#pragma unroll
                    for (int i = 0; i < kSum / 16; i++) // 16 terms: 32 bytes along a box's rows, or 16 of them
                        multiply(tmem + half * BN, a + i * (a_along_sum ? 128 : 2), b + i * (MODE == kProducts ? 128 : 2), kind, k > tile.from || i > 0);
                    when_multiplied(empty + 8 * s);
                }
                if (!fine) break;
                when_multiplied(done + 8 * half);
                m++;
            }
            if (!fine) {
                volatile int patient = 0;
                when_multiplied(drained);
                barrier_wait(drained, 0, &patient);
            }
        }
        __syncwarp();
    } else {
        const int quarter = warp & 3, side = (warp - 2) >> 2; // 32 rows, half of the columns
        const uint32_t mine = staging + (warp - 2) * 4096, my_row = mine + lane * 128;
        const uint32_t from = tmem + ((uint32_t)quarter << 21) + side * HALF;
        const float k_all = MODE == kProducts ? gradient_scale<T>(h) : 0.0f;
        uint32_t m = 0;
        for (long long t = blockIdx.x; tile_at<MODE>(p, t, rows, tile); t += gridDim.x) {
            const Product &w = p.of[tile.product];
            const bool nothing = tile.from >= tile.to;
            const uint32_t half = m & 1, at = from + half * BN;
            const int row = tile.row * 128 + quarter * 32 + lane, column = tile.column * BN + side * HALF; // (of the lane; the first)
            if (MODE != kProducts) { // the columns' bias; classes that there are not have a logit of -inf
                asm volatile("bar.sync 1, 256;" ::: "memory");
                if (threadIdx.x - 64 < BN) {
                    const int c = h.first + tile.column * BN + (int)threadIdx.x - 64;
                    s_bias[threadIdx.x - 64] = c >= h.a.classes ? -INFINITY : h.a.bias ? to_float(static_cast<const T *>(h.a.bias)[c]) : 0.0f;
                }
                asm volatile("bar.sync 1, 256;" ::: "memory");
            }
            bool fine = true;
            if (!nothing) {
                fine = barrier_wait(done + 8 * half, m / 2 & 1, s_gave_up);
                fine = __all_sync(0xffffffffu, fine);
                tmem_after_sync();
                m++;
            }
            auto give_back = [&] { // behind the last load of the tile
                if (nothing) return;
                tmem_before_sync();
                __syncwarp();
                if (lane == 0) barrier_arrive(taken + 8 * half);
            };
            const float4 *bias4 = reinterpret_cast<const float4 *>(s_bias + side * HALF);
            if constexpr (MODE == kStatistics) {
                const bool there = row < rows;
                const long long orig = !there ? 0 : h.map ? h.map[row] : row;
                Picks picks{{-1, -1}, {0.0f, 0.0f}, 0.0f, 0.0f, false, true};
                if (there) picks = picks_of(h.a, orig);
                const bool apart = h.a.smoothing > 0.0f;
                const int left = (int)h.a.classes - (h.first + column); // classes from the first column on
                float top = kLowest, sum = 0.0f, away = 0.0f;
#pragma unroll 1
                for (int c = 0; c < HALF; c += 32) {
                    uint32_t raw[32];
                    tmem_load(raw, at + c);
                    Two z[16];
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        const float4 b = bias4[(c + j) / 4];
                        z[j / 2] = add_rn(Two(__uint_as_float(raw[j]), __uint_as_float(raw[j + 1])), Two(b.x, b.y));
                        z[j / 2 + 1] = add_rn(Two(__uint_as_float(raw[j + 2]), __uint_as_float(raw[j + 3])), Two(b.z, b.w));
                    }
                    float most = top;
#pragma unroll
                    for (int j = 0; j < 16; j++) most = fmaxf(most, fmaxf(z[j].lo(), z[j].hi()));
                    sum *= exp_of(top - most);
                    if (apart) away += (float)min(c, max(left, 0)) * fmaxf(top - most, kLowest);
                    top = most;
                    const Two minus(-top, -top), log2e(kLog2e, kLog2e);
                    Two part[2] = {Two(0.0f, 0.0f), Two(0.0f, 0.0f)};
#pragma unroll
                    for (int j = 0; j < 16; j++) {
                        z[j] = add_rn(z[j], minus);
                        const Two d = mul_rn(z[j], log2e);
                        part[j & 1] = add_rn(part[j & 1], Two(exp2_of(d.lo()), exp2_of(d.hi())));
                    }
                    part[0] = add_rn(part[0], part[1]);
                    sum += part[0].lo() + part[0].hi();
                    if (apart) {
                        float all = 0.0f;
#pragma unroll
                        for (int j = 0; j < 16; j++) all += (c + 2 * j < left ? z[j].lo() : 0.0f) + (c + 2 * j + 1 < left ? z[j].hi() : 0.0f);
                        away += all;
                    }
                }
#pragma unroll
                for (int k = 0; k < 2; k++) { // the labels' logits
                    const long long c = picks.bad || picks.weight[k] == 0.0f ? -1 : picks.label[k] - h.first - column;
                    const bool wanted = c >= 0 && c < HALF;
                    for (uint32_t who = __ballot_sync(0xffffffffu, wanted); who; who &= who - 1) {
                        const int one = __ffs(who) - 1, there_c = __shfl_sync(0xffffffffu, (int)c, one);
                        const float z = tmem_load_one(at + there_c) + s_bias[side * HALF + there_c];
                        if (lane == one) h.a.stats[4 * orig + 2 + k] = fine ? z : NAN;
                    }
                }
                give_back();
                const long long part = (long long)(2 * tile.column + side) * h.rows_pad + row;
                h.parts[part] = fine ? make_float2(top, sum) : make_float2(NAN, NAN);
                if (apart) h.parts_apart[part] = away;
            } else {
                float factor = k_all, flat = 0.0f, row_top = 0.0f, held = 0.0f;
                int label[2] = {-1, -1};       // columns of the labels
                float written[2] = {0.0f, 0.0f}; // and what is there
                if constexpr (MODE == kGradient) {
                    factor = 0.0f;
                    if (row < rows) {
                        const long long orig = h.map ? h.map[row] : row;
                        const Picks picks = picks_of(h.a, orig);
                        const float4 stats = reinterpret_cast<const float4 *>(h.a.stats)[orig];
                        held = kHeld<T>;
                        if (h.a.upstream && h.a.upstream_per_row) {
                            const float most = *h.most;
                            held *= most == 0.0f ? 0.0f : h.a.upstream[orig] / most;
                        }
                        row_top = stats.x;
                        if (stats.y == 0.0f) held = 0.0f; // (no logit but -inf)
                        factor = held * picks.total * stats.y;
                        flat = held * picks.flat;
                        if (picks.bad) {
                            factor = NAN;
                        } else {
#pragma unroll
                            for (int k = 0; k < 2; k++) {
                                const long long c = picks.label[k] - h.first - column;
                                if (picks.weight[k] == 0.0f || c < 0 || c >= HALF) continue;
                                label[k] = (int)c;
                                written[k] = factor * exp_of((k ? stats.w : stats.z) - row_top) - flat - held * picks.weight[k];
                            }
                            if (label[0] >= 0 && label[0] == label[1]) {
                                written[0] -= held * picks.weight[1];
                                label[1] = -1;
                            }
                        }
                    }
                    if (!fine) factor = NAN;
                }
                const bool blank = nothing || (MODE == kGradient && row >= rows); // (what is there is no number, perhaps)
                const Two minus(-row_top, -row_top), log2e(kLog2e, kLog2e), times(factor, factor), less(-flat, -flat);
                const int row0 = tile.row * 128 + quarter * 32 + (MODE == kProducts ? tile.split * w.c_rows : 0);
                // 32 columns from c on
                auto values = [&](Two(&v)[16], int c) {
                    uint32_t raw[32];
                    tmem_load(raw, at + c);
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        Two a(__uint_as_float(raw[j]), __uint_as_float(raw[j + 1])), b(__uint_as_float(raw[j + 2]), __uint_as_float(raw[j + 3]));
                        if constexpr (MODE == kGradient) {
                            const float4 bias = bias4[(c + j) / 4];
                            a = mul_rn(add_rn(add_rn(a, Two(bias.x, bias.y)), minus), log2e);
                            b = mul_rn(add_rn(add_rn(b, Two(bias.z, bias.w)), minus), log2e);
                            a = fma_rn(Two(exp2_of(a.lo()), exp2_of(a.hi())), times, less);
                            b = fma_rn(Two(exp2_of(b.lo()), exp2_of(b.hi())), times, less);
                        } else if (w.leaves == kWritten) {
                            a = mul_rn(a, times);
                            b = mul_rn(b, times);
                        }
                        v[j / 2] = a;
                        v[j / 2 + 1] = b;
                    }
                    if (blank)
#pragma unroll
                        for (int j = 0; j < 16; j++) v[j] = Two(0.0f, 0.0f);
                    if (!fine)
#pragma unroll
                        for (int j = 0; j < 16; j++) v[j] = Two(NAN, NAN);
                };
                auto room_free = [&] {
                    if (lane == 0) boxes_read();
                    __syncwarp();
                };
                auto piece = [&](int j, uint4 v) {
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(my_row + ((j ^ (lane & 7)) << 4)), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
                };
                const int x_last = MODE == kGradient ? h.columns : (int)h.a.width;
                auto leave = [&](int x) {
                    shared_to_copies();
                    __syncwarp();
                    if (lane == 0 && x < x_last && row0 < w.c_last) {
                        if (MODE == kProducts && w.leaves == kAdded32)
                            add_box(&w.c, x, row0, mine);
                        else
                            store_box(&w.c, x, row0, mine);
                        boxes_commit();
                    }
                };
                if (MODE == kGradient || w.leaves == kWritten) {
#pragma unroll 1
                    for (int c = 0; c < HALF; c += 64) {
                        room_free();
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            Two v[16];
                            values(v, c + 32 * i);
#pragma unroll
                            for (int j = 0; j < 4; j++)
                                piece(4 * i + j, make_uint4(two_of<T>(v[4 * j].lo(), v[4 * j].hi()), two_of<T>(v[4 * j + 1].lo(), v[4 * j + 1].hi()),
                                                            two_of<T>(v[4 * j + 2].lo(), v[4 * j + 2].hi()), two_of<T>(v[4 * j + 3].lo(), v[4 * j + 3].hi())));
                        }
                        if (c + 64 >= HALF) give_back();
                        if constexpr (MODE == kGradient) {
#pragma unroll
                            for (int k = 0; k < 2; k++) {
                                const int l = label[k] - c;
                                if (label[k] < 0 || l < 0 || l >= 64) continue;
                                const uint32_t two = two_of<T>(fine ? written[k] : NAN, 0.0f);
                                asm volatile("st.shared.b16 [%0], %1;" ::"r"(my_row + ((l / 8 ^ (lane & 7)) << 4) + l % 8 * 2), "h"((uint16_t)two) : "memory");
                            }
                        }
                        leave(column + c);
                        if constexpr (MODE == kGradient) {
                            if (h.bias_parts) { // sums of these 32 rows, two columns for a lane
                                float2 s = make_float2(0.0f, 0.0f);
#pragma unroll 8
                                for (int r = 0; r < 32; r++) {
                                    uint32_t two;
                                    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(two) : "r"(mine + r * 128 + ((lane / 4 ^ (r & 7)) << 4) + lane % 4 * 4) : "memory");
                                    Pack<T, 4> pack;
                                    pack.raw = make_uint2(two, 0);
                                    float f[4];
                                    pack.get(f);
                                    s.x += f[0];
                                    s.y += f[1];
                                }
                                const int x = column + c + 2 * lane;
                                float *to = h.bias_parts + (long long)(tile.row * 4 + quarter) * w.c_rows + x;
                                if (x < w.c_rows) *reinterpret_cast<float2 *>(to) = s;
                            }
                        }
                    }
                } else {
#pragma unroll 1
                    for (int c = 0; c < HALF; c += 32) {
                        room_free();
                        Two v[16];
                        values(v, c);
#pragma unroll
                        for (int j = 0; j < 8; j++)
                            piece(j, make_uint4(__float_as_uint(v[2 * j].lo()), __float_as_uint(v[2 * j].hi()), __float_as_uint(v[2 * j + 1].lo()), __float_as_uint(v[2 * j + 1].hi())));
                        if (c + 32 >= HALF) give_back();
                        leave(column + c);
                    }
                }
            }
        }
        if (MODE != kStatistics && lane == 0) boxes_written();
    }
    tmem_before_sync();
    __syncthreads();
    tmem_after_sync();
    if (warp == 1) tmem_free(tmem, 2 * BN);
}

// Rows' statistics joined over the classes: 32 rows per CTA, whose eight warps each take every eighth part.
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ Head h) {
    __shared__ float s_part[8][3][32];
    wait_for_previous();
    let_next_begin();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, row = blockIdx.x * 32 + lane, rows = rows_counted(h);
    if (blockIdx.x * 32 >= rows) return;
    const bool apart = h.a.smoothing > 0.0f;
    const int each = h.part_columns;
    float top = kLowest, sum = 0.0f, away = 0.0f, mass = 0.0f;
#pragma unroll 4
    for (int k = warp; k < h.part_count; k += 8) {
        const long long at = (long long)k * h.rows_pad + row;
        const float2 one = h.parts[at];
        const float most = fmaxf(top, one.x);
        sum = sum * exp_of(top - most) + one.y * exp_of(one.x - most);
        if (apart) {
            const float there = (float)max(0, min(each, (int)h.a.classes - k * each));
            away = away + mass * fmaxf(top - most, kLowest) + h.parts_apart[at] + there * fmaxf(one.x - most, kLowest);
            mass += there;
        }
        top = most;
        if (one.x != one.x) sum = NAN;
    }
    s_part[warp][0][lane] = top;
    s_part[warp][1][lane] = sum;
    s_part[warp][2][lane] = away;
    __syncthreads();
    if (warp || row >= rows) return;
    float most = top;
    for (int k = 1; k < 8; k++) most = fmaxf(most, s_part[k][0][lane]);
    sum = away = 0.0f;
    for (int k = 0; k < 8; k++) {
        const float t = s_part[k][0][lane];
        sum += s_part[k][1][lane] * exp_of(t - most);
        if (!apart) continue;
        long long there = 0; // classes that the warp has joined
        for (int part = k; part < h.part_count; part += 8) there += max(0, min(each, (int)h.a.classes - part * each));
        away += s_part[k][2][lane] + (float)there * fmaxf(t - most, kLowest);
    }
    const long long orig = h.map ? h.map[row] : row;
    const Picks p = picks_of(h.a, orig);
    float4 *stats = reinterpret_cast<float4 *>(h.a.stats) + orig;
    float loss = NAN, over = NAN;
    if (!p.bad) {
        const float picked[2] = {stats->z, stats->w};
        float dot = p.flat > 0.0f ? p.flat * away : 0.0f;
        for (int k = 0; k < 2; k++)
            if (p.weight[k] != 0.0f) dot += p.weight[k] * (picked[k] - most);
        loss = sum == 0.0f ? 0.0f : p.total * logf(sum) - dot;
        over = sum == 0.0f ? 0.0f : 1.0f / sum;
    }
    h.a.row_loss[orig] = loss;
    stats->x = most;
    stats->y = over;
}

// Which rows count, in their order: the place of each, or -1; a row for each place.  One CTA; rows that do not count get a loss of 0.
__global__ void __launch_bounds__(1024) places_kernel(const __grid_constant__ ffcvb_linear_cross_entropy_args a, int *map, int *place, float *counted) {
    __shared__ int s_count[33];
    wait_for_previous();
    let_next_begin();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t *labels = static_cast<const int64_t *>(a.target);
    // a warp has a run of rows, 32 at a time
    const int run = (int)((a.rows + 1023) / 1024) * 32, first = warp * run, last = min(first + run, (int)a.rows);
    int n = 0;
    for (int r = first + lane; r < last; r += 32) n += labels[r * a.target_stride] != a.ignore_index;
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) s_count[warp] = n;
    __syncthreads();
    int before = __reduce_add_sync(0xffffffffu, lane < warp ? s_count[lane] : 0);
    for (int r0 = first; r0 < last; r0 += 32) {
        const int r = r0 + lane;
        const bool counts = r < last && labels[r * a.target_stride] != a.ignore_index;
        const uint32_t those = __ballot_sync(0xffffffffu, counts);
        const int here = before + __popc(those & ((1u << lane) - 1));
        if (counts) map[here] = r;
        if (r < last) {
            place[r] = counts ? here : -1;
            if (!counts && !a.from_stats) {
                if (a.row_loss) a.row_loss[r] = 0.0f;
                reinterpret_cast<float4 *>(a.stats)[r] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
        }
        before += __popc(those);
    }
    if (warp == 31 && lane == 0) *counted = (float)before;
}

// Rows of `width` values of 16 bits in places that the copies can begin at; rows behind those that count, up to the next 128, and columns behind
// the last one are 0.
__global__ void __launch_bounds__(256) lay_kernel(const uint16_t *__restrict__ from, long long stride, int rows, int width, const int *map, const float *counted,
                                                  uint16_t *__restrict__ to, int pad, int wide) {
    wait_for_previous();
    let_next_begin();
    if (counted) rows = (int)*counted;
    const int all = (rows + 127) / 128 * 128, packs = pad / 8;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < (long long)all * packs; i += (long long)gridDim.x * 256) {
        const int r = (int)(i / packs), c = (int)(i % packs) * 8;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (r < rows) {
            const uint16_t *at = from + (map ? map[r] : r) * stride + c;
            if (wide && c + 8 <= width) {
                v = *reinterpret_cast<const uint4 *>(at);
            } else {
                uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (c + j < width) w[j / 2] |= (uint32_t)at[j] << (16 * (j & 1));
                v = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
        *reinterpret_cast<uint4 *>(to + (long long)r * pad + c) = v;
    }
}

// The largest size of the rows' upstream gradients.
__global__ void __launch_bounds__(1024) most_kernel(const float *__restrict__ upstream, long long rows, float *most) {
    __shared__ float s_most[32];
    wait_for_previous();
    let_next_begin();
    float m = 0.0f;
    bool bad = false;
    for (long long i = threadIdx.x; i < rows; i += 1024) {
        const float v = fabsf(upstream[i]);
        bad |= v != v;
        m = fmaxf(m, v);
    }
    m = warp_max(m);
    if ((threadIdx.x & 31) == 0) s_most[threadIdx.x >> 5] = m;
    bad = __syncthreads_or(bad);
    if (threadIdx.x < 32) {
        m = warp_max(s_most[threadIdx.x]);
        if (threadIdx.x == 0) *most = bad ? NAN : m;
    }
}

// Gradients from parts of sums in 32 bits, or of rows that count from 16 bits: out[r] = sum of parts[place of r]; rows without a place are 0.
template <typename T, typename Part>
__global__ void __launch_bounds__(256) settle_kernel(const __grid_constant__ Head h, const Part *__restrict__ parts, long long part_size, int splits, int pad, const int *place,
                                                     T *__restrict__ out, int rows, int width) {
    wait_for_previous();
    let_next_begin();
    const float k = sizeof(Part) == 4 ? gradient_scale<T>(h) : 1.0f;
    const int packs = (width + 7) / 8;
    const bool wide = width % 8 == 0;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < (long long)rows * packs; i += (long long)gridDim.x * 256) {
        const int r = (int)(i / packs), c = (int)(i % packs) * 8, from = place ? place[r] : r;
        float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
        if (from >= 0) {
            const Part *at = parts + (long long)from * pad + c;
            for (int s = 0; s < splits; s++, at += part_size) {
                constexpr int N = kWide<Part>;
#pragma unroll
                for (int j = 0; j < 8; j += N) {
                    Pack<Part, N> pack;
                    float f[N];
                    pack.load(at + j);
                    pack.get(f);
#pragma unroll
                    for (int l = 0; l < N; l++) v[j + l] += f[l];
                }
            }
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] *= k;
        }
        T *to = out + (long long)r * width + c;
        if (wide) {
            Pack<T, 8> pack;
            pack.set(v);
            pack.store(to);
        } else {
            for (int j = 0; j < 8 && c + j < width; j++) to[j] = from_float<T>(v[j]);
        }
    }
}

// The bias' gradient: sums over 32 rows each added up, 32 columns per CTA.
template <typename T>
__global__ void __launch_bounds__(256) bias_kernel(const __grid_constant__ Head h, int pad) {
    __shared__ float s_sum[8][32];
    wait_for_previous();
    let_next_begin();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    const int parts = (rows_counted(h) + 127) / 128 * 4;
    float sum = 0.0f;
    if (c < h.columns) {
#pragma unroll 8
        for (int k = warp; k < parts; k += 8) sum += h.bias_parts[(long long)k * pad + c];
    }
    s_sum[warp][lane] = sum;
    __syncthreads();
    if (warp || c >= h.columns) return;
    for (int k = 1; k < 8; k++) sum += s_sum[k][lane];
    static_cast<T *>(h.a.grad_bias)[h.first + c] = from_float<T>(sum * gradient_scale<T>(h));
}

// ---- the host's part -------------------------------------------------------------------------------------------------

inline int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// A gradient product: how its tiles are cut, and how it leaves.
struct Cut {
    int splits = 1;
    bool direct = true;
};

// What a call does, and where in the workspace (offsets in bytes).
struct Plan {
    int64_t rows_pad, width_pad, chunk, chunks;  // (classes at once)
    bool counted, lay_hidden, lay_weight, grads, hidden_grad, weight_grad, bias_grad;
    int stat_columns, sum_columns;               // BN
    Cut of_hidden, of_weight;
    int64_t map, place, count, most, hidden, weight, parts, apart, grad, hidden_parts, hidden_rows, weight_parts, bias_parts, bytes;
};

// G's bytes at most.  (So many classes at once that dw's tiles and the sum over classes fill the GPU; 8 GB of HBM would hold 32 times as much.)
constexpr int64_t kMostGradient = 256ll << 20;

bool aligned(const void *p, int64_t stride) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride % 8 == 0; }

// Tiles of a product, and parts of its sum where there are too few of them: parts of at least eight blocks.
Cut cut_of(int64_t tiles, int64_t others, int64_t blocks, bool direct) {
    Cut cut;
    if (tiles > 0 && tiles + others < kSms && blocks >= 16) cut.splits = (int)std::min<int64_t>(blocks / 8, std::max<int64_t>(1, kSms / (tiles + others)));
    cut.direct = direct && cut.splits == 1;
    return cut;
}

Plan plan_of(const ffcvb_linear_cross_entropy_args &a) {
    Plan p{};
    p.rows_pad = up(a.rows, 128);
    p.width_pad = up(a.width, 8);
    p.counted = a.has_ignore && a.target_kind == FFCVB_TARGET_LABELS;
    p.lay_hidden = p.counted || !aligned(a.hidden, a.hidden_stride);
    p.lay_weight = !aligned(a.weight, a.weight_stride);
    p.hidden_grad = a.grad_hidden, p.weight_grad = a.grad_weight, p.bias_grad = a.grad_bias;
    p.grads = p.hidden_grad || p.weight_grad || p.bias_grad;
    const int64_t row_tiles = p.rows_pad / 128;
    p.stat_columns = row_tiles * ((a.classes + 255) / 256) < kSms ? 128 : 256;
    p.chunks = (a.classes * p.rows_pad * 2 + kMostGradient - 1) / kMostGradient;
    p.chunk = up((a.classes + p.chunks - 1) / p.chunks, 256);
    p.chunks = (a.classes + p.chunk - 1) / p.chunk;
    // columns of the gradients' tiles: those that need the fewer steps
    auto cost = [&](int64_t bn) {
        const int64_t tiles = (row_tiles + p.chunk / 128) * ((a.width + bn - 1) / bn);
        return (tiles + kSms - 1) / kSms * bn;
    };
    p.sum_columns = cost(128) < cost(256) ? 128 : 256;
    const int64_t column_tiles = (a.width + p.sum_columns - 1) / p.sum_columns;
    const int64_t hidden_tiles = p.hidden_grad ? row_tiles * column_tiles : 0, weight_tiles = p.weight_grad ? p.chunk / 128 * column_tiles : 0;
    p.of_hidden = cut_of(hidden_tiles, weight_tiles, p.chunk / kSum, p.chunks == 1 && (p.counted || a.width % 8 == 0));
    p.of_weight = cut_of(weight_tiles, hidden_tiles, (a.rows + kSum - 1) / kSum, a.width % 8 == 0);
    int64_t at = 0;
    auto take = [&](bool wanted, int64_t bytes) {
        const int64_t here = at;
        if (wanted) at += up(bytes, 256);
        return here;
    };
    p.map = take(p.counted, p.rows_pad * 4);
    p.place = take(p.counted, p.rows_pad * 4);
    p.count = take(p.counted, 4);
    p.most = take(a.upstream && a.upstream_per_row, 4);
    p.hidden = take(p.lay_hidden, p.rows_pad * p.width_pad * 2);
    p.weight = take(p.lay_weight, up(a.classes, 128) * p.width_pad * 2);
    const int64_t parts = up(a.classes, p.stat_columns) / (p.stat_columns / 2) * p.rows_pad;
    p.parts = take(!a.from_stats, parts * 8);
    p.apart = take(!a.from_stats && a.smoothing > 0.0f, parts * 4);
    p.grad = take(p.grads, p.rows_pad * p.chunk * 2);
    const int64_t wide = up(a.width, 32); // (boxes of 32 values)
    p.hidden_parts = take(p.hidden_grad && !p.of_hidden.direct, p.of_hidden.splits * p.rows_pad * wide * 4);
    p.hidden_rows = take(p.hidden_grad && p.of_hidden.direct && p.counted, p.rows_pad * p.width_pad * 2);
    p.weight_parts = take(p.weight_grad && !p.of_weight.direct, p.of_weight.splits * p.chunk * wide * 4);
    p.bias_parts = take(p.bias_grad, p.rows_pad / 32 * p.chunk * 4);
    p.bytes = at;
    return p;
}

const char *wrong(const ffcvb_linear_cross_entropy_args &a) {
    if (a.type != FFCVB_TYPE_F16 && a.type != FFCVB_TYPE_BF16) return "values must be of 16 bits";
    if (a.rows < 0 || a.classes < 1 || a.width < 1 || a.rows > 1 << 24 || a.classes > 1 << 24 || a.width > 1 << 16) return "bad size";
    if (a.hidden_stride < 0 || a.weight_stride < 0 || (a.rows > 1 && a.hidden_stride < a.width) || (a.classes > 1 && a.weight_stride < a.width)) return "bad stride";
    if (a.target_kind != FFCVB_TARGET_LABELS && a.target_kind != FFCVB_TARGET_MIXED) return "bad target";
    if (!(a.smoothing >= 0.0f && a.smoothing <= 1.0f) || (a.has_ignore && a.target_kind != FFCVB_TARGET_LABELS)) return "bad argument";
    if (a.rows > 0 && (!a.hidden || !a.weight || !a.target || !a.stats || (!a.from_stats && !a.row_loss))) return "an address is missing";
    if (a.from_stats && !a.grad_hidden && !a.grad_weight && !a.grad_bias) return "nothing to do";
    if (a.grad_bias && !a.bias) return "no bias";
    return nullptr;
}

template <int MODE, typename T, int BN> bool launch_products(const Products &p, int64_t tiles, cudaStream_t stream) {
    auto *kernel = products_kernel<MODE, T, BN>;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kRoom<BN>) != cudaSuccess) return false;
    return launch_early(kernel, (unsigned)std::min<int64_t>(tiles, kSms), kThreads, kRoom<BN>, stream, p) == cudaSuccess;
}
template <int MODE, typename T> bool launch_products(int columns, const Products &p, int64_t tiles, cudaStream_t stream) {
    return columns == 256 ? launch_products<MODE, T, 256>(p, tiles, stream) : launch_products<MODE, T, 128>(p, tiles, stream);
}

template <typename T> int run(const ffcvb_linear_cross_entropy_args &a, uint8_t *room, cudaStream_t st) {
    const Plan p = plan_of(a);
    const int type = a.type;
    const int64_t row_tiles = p.rows_pad / 128;
    auto at = [&](int64_t offset) { return static_cast<void *>(room + offset); };
    Products g{};
    Head &h = g.head;
    h.a = a;
    h.rows_pad = (int)p.rows_pad;
    h.map = p.counted ? static_cast<int *>(at(p.map)) : nullptr;
    h.place = p.counted ? static_cast<int *>(at(p.place)) : nullptr;
    h.counted = p.counted ? static_cast<float *>(at(p.count)) : nullptr;
    h.most = static_cast<float *>(at(p.most));
    h.parts = static_cast<float2 *>(at(p.parts));
    h.parts_apart = static_cast<float *>(at(p.apart));
    h.part_columns = p.stat_columns / 2;
    h.part_count = (int)(up(a.classes, p.stat_columns) / h.part_columns);
    if (p.counted) launch_early(places_kernel, 1, 1024, 0, st, a, static_cast<int *>(at(p.map)), static_cast<int *>(at(p.place)), static_cast<float *>(at(p.count)));
    auto lay = [&](const void *from, int64_t stride, int64_t rows, const int *map, const float *counted, void *to) {
        const unsigned ctas = (unsigned)std::min<int64_t>((up(rows, 128) * (p.width_pad / 8) + 255) / 256, kSms * 8);
        launch_early(lay_kernel, ctas, 256, 0, st, static_cast<const uint16_t *>(from), (long long)stride, (int)rows, (int)a.width, map, counted, static_cast<uint16_t *>(to),
                     (int)p.width_pad, (int)aligned(from, stride));
    };
    const void *hidden = a.hidden, *weight = a.weight;
    int64_t hidden_stride = a.hidden_stride, weight_stride = a.weight_stride, hidden_rows = a.rows;
    if (p.lay_hidden) {
        lay(a.hidden, a.hidden_stride, a.rows, h.map, h.counted, at(p.hidden));
        hidden = at(p.hidden), hidden_stride = p.width_pad, hidden_rows = p.rows_pad;
    }
    if (p.lay_weight) {
        lay(a.weight, a.weight_stride, a.classes, nullptr, nullptr, at(p.weight));
        weight = at(p.weight), weight_stride = p.width_pad;
    }
    if (a.rows == 1 || hidden_stride < p.width_pad) hidden_stride = p.width_pad;   // (one row)
    if (a.classes == 1 || weight_stride < p.width_pad) weight_stride = p.width_pad; // (one class)
    bool mapped = true, fine = true;
    const int sum_blocks = (int)((a.width + kSum - 1) / kSum);
    // logits: columns of a tile, classes from `first` on
    auto logits = [&](int columns, int64_t first, int64_t count) {
        Product &w = g.of[0];
        mapped &= matrix_map(&w.a, type, hidden, hidden_rows, a.width, hidden_stride, 128);
        mapped &= matrix_map(&w.b, type, weight, a.classes, a.width, weight_stride, columns);
        w.row_tiles = (int)row_tiles;
        w.column_tiles = (int)((count + columns - 1) / columns);
        w.sum_blocks = sum_blocks;
        w.splits = 1;
        w.a_along_sum = 0;
        w.counted = p.counted ? kRowsCounted : kFixed;
        w.b_first = (int)first;
        g.count = 1;
        h.first = (int)first;
        h.columns = (int)count;
        return row_tiles * w.column_tiles;
    };
    if (!a.from_stats) {
        const int64_t tiles = logits(p.stat_columns, 0, a.classes);
        if (!mapped) return training_fail(FFCVB_E_CUDA, "ffcvb_linear_cross_entropy: no map of a matrix");
        g.of[0].b_first = 0;
        fine &= launch_products<kStatistics, T>(p.stat_columns, g, tiles, st);
        launch_early(join_kernel, (unsigned)(p.rows_pad / 32), 256, 0, st, h);
        if (a.loss) launch_mean(a.row_loss, a.rows, h.counted, a.mean, a.loss, st);
    }
    if (!p.grads) return fine ? launched("ffcvb_linear_cross_entropy") : training_fail(FFCVB_E_CUDA, "ffcvb_linear_cross_entropy: %s", cudaGetErrorString(cudaGetLastError()));
    if (a.upstream && a.upstream_per_row) launch_early(most_kernel, 1, 1024, 0, st, a.upstream, a.rows, static_cast<float *>(at(p.most)));
    const int64_t wide = up(a.width, 32);
    auto ctas_for = [&](int64_t rows) { return (unsigned)std::min<int64_t>((rows * ((a.width + 7) / 8) + 255) / 256, kSms * 8); };
    for (int64_t chunk = 0; chunk < p.chunks; chunk++) {
        const int64_t first = chunk * p.chunk, count = std::min(p.chunk, a.classes - first);
        const int columns = row_tiles * ((count + 255) / 256) < kSms ? 128 : 256;
        int64_t tiles = logits(columns, first, count);
        mapped &= matrix_map(&g.of[0].c, type, at(p.grad), p.counted ? p.rows_pad : a.rows, count, p.chunk, 32);
        g.of[0].c_rows = (int)p.chunk; // (of the bias' sums: columns)
        g.of[0].c_last = (int)(p.counted ? p.rows_pad : a.rows);
        h.bias_parts = p.bias_grad ? static_cast<float *>(at(p.bias_parts)) : nullptr;
        if (!mapped) break;
        fine &= launch_products<kGradient, T>(columns, g, tiles, st);
        if (p.bias_grad) launch_early(bias_kernel<T>, (unsigned)((count + 31) / 32), 256, 0, st, h, (int)p.chunk);
        const int column_tiles = (int)((a.width + p.sum_columns - 1) / p.sum_columns);
        g.count = 0;
        tiles = 0;
        if (p.hidden_grad) {
            Product &w = g.of[g.count++];
            mapped &= matrix_map(&w.a, type, at(p.grad), p.counted ? p.rows_pad : a.rows, count, p.chunk, 128);
            mapped &= matrix_map(&w.b, type, weight, a.classes, a.width, weight_stride, kSum);
            if (!p.of_hidden.direct)
                mapped &= matrix_map(&w.c, FFCVB_TYPE_F32, at(p.hidden_parts), p.of_hidden.splits * p.rows_pad, wide, wide, 32);
            else if (p.counted)
                mapped &= matrix_map(&w.c, type, at(p.hidden_rows), p.rows_pad, a.width, p.width_pad, 32);
            else
                mapped &= matrix_map(&w.c, type, a.grad_hidden, a.rows, a.width, a.width, 32);
            w.row_tiles = (int)row_tiles;
            w.column_tiles = column_tiles;
            w.sum_blocks = (int)((count + kSum - 1) / kSum);
            w.splits = p.of_hidden.splits;
            w.a_along_sum = 0;
            w.leaves = p.of_hidden.direct ? kWritten : chunk ? kAdded32 : kWritten32;
            w.counted = p.counted ? kRowsCounted : kFixed;
            w.b_first = (int)first;
            w.c_rows = (int)p.rows_pad;
            w.c_last = (int)(!p.of_hidden.direct ? p.of_hidden.splits * p.rows_pad : p.counted ? p.rows_pad : a.rows);
            tiles += row_tiles * column_tiles * w.splits;
        }
        if (p.weight_grad) {
            Product &w = g.of[g.count++];
            mapped &= matrix_map(&w.a, type, at(p.grad), p.counted ? p.rows_pad : a.rows, count, p.chunk, kSum);
            mapped &= matrix_map(&w.b, type, hidden, hidden_rows, a.width, hidden_stride, kSum);
            if (p.of_weight.direct)
                mapped &= matrix_map(&w.c, type, static_cast<T *>(a.grad_weight) + first * a.width, count, a.width, a.width, 32);
            else
                mapped &= matrix_map(&w.c, FFCVB_TYPE_F32, at(p.weight_parts), p.of_weight.splits * p.chunk, wide, wide, 32);
            w.row_tiles = (int)((count + 127) / 128);
            w.column_tiles = column_tiles;
            w.sum_blocks = (int)((a.rows + kSum - 1) / kSum);
            w.splits = p.of_weight.splits;
            w.a_along_sum = 1;
            w.leaves = p.of_weight.direct ? kWritten : kWritten32;
            w.counted = p.counted ? kSumCounted : kFixed;
            w.b_first = 0;
            w.c_rows = (int)p.chunk;
            w.c_last = (int)(p.of_weight.direct ? count : p.of_weight.splits * p.chunk);
            tiles += (int64_t)w.row_tiles * column_tiles * w.splits;
        }
        if (!mapped) break;
        if (g.count) fine &= launch_products<kProducts, T>(p.sum_columns, g, tiles, st);
        if (p.weight_grad && !p.of_weight.direct)
            launch_early(settle_kernel<T, float>, ctas_for(count), 256, 0, st, h, static_cast<const float *>(at(p.weight_parts)), (long long)(p.chunk * wide),
                         p.of_weight.splits, (int)wide, (const int *)nullptr, static_cast<T *>(a.grad_weight) + first * a.width, (int)count, (int)a.width);
    }
    if (!mapped) return training_fail(FFCVB_E_CUDA, "ffcvb_linear_cross_entropy: no map of a matrix");
    if (p.hidden_grad && !p.of_hidden.direct)
        launch_early(settle_kernel<T, float>, ctas_for(a.rows), 256, 0, st, h, static_cast<const float *>(at(p.hidden_parts)), (long long)(p.rows_pad * wide), p.of_hidden.splits,
                     (int)wide, h.place, static_cast<T *>(a.grad_hidden), (int)a.rows, (int)a.width);
    else if (p.hidden_grad && p.counted)
        launch_early(settle_kernel<T, T>, ctas_for(a.rows), 256, 0, st, h, static_cast<const T *>(at(p.hidden_rows)), 0ll, 1, (int)p.width_pad, h.place,
                     static_cast<T *>(a.grad_hidden), (int)a.rows, (int)a.width);
    return fine ? launched("ffcvb_linear_cross_entropy") : training_fail(FFCVB_E_CUDA, "ffcvb_linear_cross_entropy: %s", cudaGetErrorString(cudaGetLastError()));
}

} // namespace

bool matrix_map(CUtensorMap *map, int type, const void *at, int64_t rows, int64_t cols, int64_t stride, int box) {
    using Encode = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *, const cuuint32_t *,
                                CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const Encode encode = [] {
        void *found = nullptr;
        cudaDriverEntryPointQueryResult how;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &found, 12000, cudaEnableDefault, &how) != cudaSuccess || how != cudaDriverEntryPointSuccess) found = nullptr;
        return reinterpret_cast<Encode>(found);
    }();
    if (!encode) return false;
    const int size = type_size(type);
    const cuuint64_t sizes[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)(stride * size)};
    const cuuint32_t boxes[2] = {(cuuint32_t)(128 / size), (cuuint32_t)box}, steps[2] = {1, 1};
    const CUtensorMapDataType kind = type == FFCVB_TYPE_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                     : type == FFCVB_TYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                              : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    return encode(map, kind, 2, const_cast<void *>(at), sizes, strides, boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

} // namespace ffcvb

using namespace ffcvb;

extern "C" int64_t ffcvb_linear_cross_entropy_workspace(const ffcvb_linear_cross_entropy_args *args) {
    return !args || wrong(*args) || args->rows == 0 ? 0 : plan_of(*args).bytes;
}

extern "C" int ffcvb_linear_cross_entropy(const ffcvb_linear_cross_entropy_args *args, void *workspace, void *stream) {
    if (!args) return training_fail(FFCVB_E_ARG, "ffcvb_linear_cross_entropy: no arguments");
    const ffcvb_linear_cross_entropy_args &a = *args;
    if (const char *what = wrong(a)) return training_fail(FFCVB_E_ARG, "ffcvb_linear_cross_entropy: %s", what);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a.rows > 0 && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255))) return training_fail(FFCVB_E_ARG, "ffcvb_linear_cross_entropy: no workspace");
    OnDevice here(a.device);
    // (a thread that has made no call of the runtime yet, as autograd's, has no context, without which the driver makes no maps)
    if (!here.ok() || cudaSetDevice(a.device) != cudaSuccess) return training_fail(FFCVB_E_NODEVICE, "ffcvb_linear_cross_entropy: no device %d", a.device);
    if (a.rows == 0) { // nothing but zeros
        if (a.loss && !a.from_stats) cudaMemsetAsync(a.loss, 0, 4, st);
        if (a.grad_weight) cudaMemsetAsync(a.grad_weight, 0, (size_t)(a.classes * a.width * 2), st);
        if (a.grad_bias) cudaMemsetAsync(a.grad_bias, 0, (size_t)(a.classes * 2), st);
        return launched("ffcvb_linear_cross_entropy");
    }
    return a.type == FFCVB_TYPE_F16 ? run<__half>(a, static_cast<uint8_t *>(workspace), st) : run<__nv_bfloat16>(a, static_cast<uint8_t *>(workspace), st);
}
