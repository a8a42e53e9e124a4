// Cross entropy of a linear layer's outputs, which are not kept, with the gradients of what goes in (sm_100a).
//
// With hidden values x [rows, width], weights w [classes, width] and a bias b the logits are z = x w^T + b, a row's loss is S lse(z) - sum T z
// (see cross_entropy.cu) and G = S exp(z - lse) - T the gradient of its logits; then dx = G w, dw = G^T x, db = sum of G's rows.  All are
// matrix products on the tensor cores with sums of 32 bits: x w^T a first time, whose tiles never leave the SM: of 128 logits of a row the
// largest and the sum of exponentials relative to it are left; joined, they give the loss and lse.  Then x w^T a second time, whose
// tiles leave as G, rounded to 16 bits (one rounding of at most 2^-8 (bf16) of a value that is multiplied and added with thousands of others), for as many
// classes at once as 256 MB hold (256 classes of all rows at least); of these dx's part is added up and dw's rows are finished.  So 8 * rows * classes * width
// operations instead of 6 are done, and no logits are kept; the first time leaves 8 bytes (12 with smoothing) for 128 logits of a row, or for 64 with narrow tiles.
//
// What bounds it: the tensor cores, and in long runs the clock that their power leaves.  8192 x 21841 x 1024 in bf16 with all gradients takes 1.04 ms in a short run and
// 1.2 to 1.26 in a long one; 880 us is the 8 * rows * classes * width at the rate of a large library product, 660 the 6.  Of it the statistics take 236 us (1550 TFLOP/s), the
// joining 9, and each of the two chunks of 10921 classes 130 for G (1410; 142 with the bias' sums), 240 for its products (1530) and 10 for what is left of them.  Kept in 16 bits
// instead the logits would be 358 MB written and read, and rounded before the exponentials.  64 x 1000 x 384 takes 29 to 32 us: six launches, which wait for one another.
#include "losses.h"
#include "tensor.h"

#include <algorithm>

namespace ffcvb {

namespace {

constexpr int kThreads = 320; // a warp that copies, one that multiplies, eight that take the results
constexpr int kSum = 64;      // of the sum's terms in a stage: 128 bytes
constexpr uint32_t kRowsBytes = 128 * 128, kStagingBytes = 8 * 4096;
// (of a pair's 256 columns each CTA has 128)
template <int BN, bool PAIR> constexpr uint32_t kStageBytes = kRowsBytes + (PAIR ? BN / 2 : BN) * 128;
template <int BN, bool PAIR> constexpr int kStages = 6 * 32768 / kStageBytes<BN, PAIR>;
// stages, the eight warps' staging, the bias of a tile, barriers; and what it takes to begin on 1024 bytes
template <int BN, bool PAIR> constexpr uint32_t kRoom = kStages<BN, PAIR> * kStageBytes<BN, PAIR> + kStagingBytes + 1024 + 256 + 1024;

enum { kStatistics, kGradient, kProducts };      // what a kernel makes of its products
enum { kWritten, kWritten32, kAdded32 };         // how products leave: as they are to be, or in 32 bits
enum { kFixed, kRowsCounted, kSumCounted };      // what depends on the number of rows that count

// One product A B of matrices, in tiles of 128, or a pair's 256, by BN.
struct alignas(64) Product {
    CUtensorMap a, b, c;
    void *out;           // what C is a map of (kProducts)
    int64_t out_stride;
    int row_tiles, column_tiles, sum_blocks;
    int a_along_sum;     // A's rows in memory run along the sum
    int leaves, counted;
    int b_first;         // where B begins along the sum (kProducts), or its rows (else)
    int c_last;          // C's rows
    int unused[4];
};

struct Head {
    ffcvb_linear_cross_entropy_args a;
    const int *map;      // rows that count, or NULL: all
    const int *place;    // a row's place among them, or -1
    const float *counted;
    float2 *parts;       // [classes / part_columns][rows_pad]: largest logit and sum of exponentials
    float *parts_apart;  // the same: `share` times the sum of logits relative to the largest; with smoothing
    float *bias_parts;   // [rows_pad / 32][chunk]
    const float *most;   // largest upstream of a row that counts
    // What smoothing gives every class of the target.  (It multiplies differences before they are added up: a sum of those to logits of the type's lowest value, which mask
    // classes, would not be finite, the loss is.)
    float share;
    int rows_pad, first, columns; // classes of this chunk
    int part_count, part_columns, chunk;
};

// Products that one launch makes.  The blocks of all tiles' sums, in their order, are dealt out to the CTAs in equal runs, so that all end at once; what a CTA
// has of a tile that is not its own alone it leaves as a part in 32 bits, the first one of its run or the last.
struct Products {
    Product of[2];
    CUtensorMap part;    // [2 * CTAs * 128, BN]
    const float *parts;
    int count, units, lanes; // (units: CTAs or pairs)
    int high;                // rows of a tile
    int unused[10];
    Head head;
};

// G, whose values are at most 1 with targets that are shares, is held times this: in fp16 those of less than 2^-24 would be lost.
template <typename T> constexpr float kHeld = 1.0f;
template <> constexpr float kHeld<__half> = 16384.0f;

template <typename T> __device__ __forceinline__ uint32_t two_of(float lo, float hi);
template <> __device__ __forceinline__ uint32_t two_of<__half>(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
}
template <> __device__ __forceinline__ uint32_t two_of<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
}

// Sums over a warp's rows, a row per lane, of two times 32 columns; a lane gets its column's of either.  Lanes exchange halves of what they have left, in 31 shuffles for 32 columns.
// (1021 x 21841 x 768 136 us with them, 139 with 32 columns at a time, 142 by way of shared memory in 32 bits, 135 where the rounded boxes were read back, 131 without a bias;
// 16384 x 21841 x 128 962, 1012, 1036, 932 and 880.)
__device__ __forceinline__ void sum_rows(Two (&v)[2][16], float (&sum)[2]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int turn = 0; turn < 4; turn++) {
        const int n = 8 >> turn;
        const bool upper = lane & 2 * n;
#pragma unroll
        for (int j = 0; j < n; j++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const Two keep = upper ? v[i][j + n] : v[i][j], give = upper ? v[i][j] : v[i][j + n];
                v[i][j] = add_rn(keep, Two(__shfl_xor_sync(0xffffffffu, give.lo(), 2 * n), __shfl_xor_sync(0xffffffffu, give.hi(), 2 * n)));
            }
    }
    const bool upper = lane & 1;
#pragma unroll
    for (int i = 0; i < 2; i++) sum[i] = (upper ? v[i][0].hi() : v[i][0].lo()) + __shfl_xor_sync(0xffffffffu, upper ? v[i][0].lo() : v[i][0].hi(), 1);
}

__device__ __forceinline__ int rows_counted(const Head &h) { return h.counted ? (int)*h.counted : (int)h.a.rows; }

// What all gradients are multiplied by behind the sums.
template <typename T> __device__ __forceinline__ float gradient_scale(const Head &h) {
    float k = h.a.scale / kHeld<T>;
    if (h.a.upstream) k *= h.a.upstream_per_row ? *h.most : *h.a.upstream;
    if (h.a.mean) k /= h.counted ? fmaxf(*h.counted, 1.0f) : (float)h.a.rows;
    return k;
}

// A tile, or a run of its sum: of which product and where; whether it is the whole.
struct Tile {
    int product, row, column, from, to;
    bool whole;
};
__device__ __forceinline__ int row_tiles_of(const Products &p, const Product &w, int rows) { return w.counted == kRowsCounted ? (rows + p.high - 1) / p.high : w.row_tiles; }
// (a sum without terms is one block long, all the same)
__device__ __forceinline__ int sum_blocks_of(const Product &w, int rows) { return w.counted == kSumCounted ? max(1, (rows + kSum - 1) / kSum) : w.sum_blocks; }
// Blocks of runs, at least: shorter ones cost more than they save.  (As built then, 64 x 1000 x 384 33 us, 42 with 1, 41 with 16; 4096 x 100 x 384 54, 67 and 58; 2048 x 1000 x 768
// 54, 54 and 49; larger ones within one in a hundred.)
constexpr int kLeastRun = 4;
// How blocks are dealt out: with few columns of tiles those of each column, in the same way to as many CTAs or pairs, so that those with the same rows read A at the same time;
// else of all tiles, those of the same columns one after another.  (The products of 8192 x 10921 x 1024, four columns: 240 us, 450 where neighbouring CTAs read different
// rows; 2048 x 8000 x 2560, ten columns: 246 us in all, 251 with all tiles in a line.)
struct Runs {
    int lanes, all, units; // columns that are dealt out apart; blocks, and CTAs or pairs with a run, of each
    int each, more;       // blocks of a run, and runs with one more
    __device__ __forceinline__ Runs(const Products &p, int rows) : lanes(p.lanes), all(0) {
        for (int i = 0; i < p.count; i++) all += row_tiles_of(p, p.of[i], rows) * sum_blocks_of(p.of[i], rows);
        if (lanes == 1) all *= p.of[0].column_tiles;
        units = min(p.units / lanes, max(1, all / kLeastRun));
        each = all / units;
        more = all - each * units;
    }
    __device__ __forceinline__ int begin(int n) const { return each * n + min(n, more); }
    __device__ __forceinline__ int lane(int unit) const { return unit % lanes; }
    __device__ __forceinline__ int place(int unit) const { return unit / lanes; }
};
// The tile that block `at` of a lane's is in, from that block on.
__device__ __forceinline__ Tile tile_of(const Products &p, const Runs &runs, int lane, int at, int rows) {
    Tile tile;
    tile.product = 0;
    const int columns = runs.lanes == 1 ? p.of[0].column_tiles : 1;
    if (p.count > 1) {
        const int here = row_tiles_of(p, p.of[0], rows) * sum_blocks_of(p.of[0], rows) * columns;
        if (at >= here) at -= here, tile.product = 1;
    }
    const Product &w = p.of[tile.product];
    const int blocks = sum_blocks_of(w, rows), row_tiles = row_tiles_of(p, w, rows), t = at / blocks;
    tile.from = at - t * blocks;
    tile.to = blocks;
    tile.column = columns == 1 ? 0 : t / row_tiles;
    tile.row = t - tile.column * row_tiles;
    if (runs.lanes > 1) tile.column = lane;
    tile.whole = tile.from == 0;
    return tile;
}
// A CTA's tiles one after another.
template <int MODE> struct Walk {
    long long at, end;
    int step;
    __device__ __forceinline__ Walk(const Products &p, int rows, int unit) : step(p.units) {
        at = unit;
        end = (long long)row_tiles_of(p, p.of[0], rows) * p.of[0].column_tiles;
    }
    __device__ __forceinline__ bool next(const Products &p, int rows, Tile &tile) { // tiles of the same weights one after another
        if (at >= end) return false;
        const int row_tiles = row_tiles_of(p, p.of[0], rows), column = (int)(at / row_tiles);
        tile = Tile{0, (int)(at - (long long)column * row_tiles), column, 0, p.of[0].sum_blocks, true};
        at += step;
        return true;
    }
};
template <> struct Walk<kProducts> {
    Runs runs;
    int lane, at, end;
    __device__ __forceinline__ Walk(const Products &p, int rows, int unit) : runs(p, rows) {
        const int place = runs.place(unit);
        lane = runs.lane(unit);
        at = place < runs.units ? runs.begin(place) : 0;
        end = place < runs.units ? runs.begin(place + 1) : 0;
    }
    __device__ __forceinline__ bool next(const Products &p, int rows, Tile &tile) {
        if (at >= end) return false;
        tile = tile_of(p, runs, lane, at, rows);
        if (end - at < tile.to - tile.from) {
            tile.to = tile.from + end - at;
            tile.whole = false;
        }
        at += tile.to - tile.from;
        return true;
    }
};

// A CTA per SM that takes tile after tile.  Products of the next tile go into the other half of TMEM while eight warps, two for each 32 rows, take
// the last one's.  A wait that does not end makes the CTA give up: all that it has not finished is NaN, and it ends.
//
// A CTA of a pair copies its own 128 rows of A and half of the columns of B, 32 KB for 64 terms, and the first one's instruction multiplies both: half of the
// shared memory's traffic for B.  (8192 x 10921 x 1024: products 240 us, 263 by single CTAs.)  Six stages of 32 KB, 192 KB, leave room for 32 KB of results, which
// leave as boxes of 32 rows by 128 bytes; written by the threads themselves G takes 140 us instead of 128.  For the statistics a thread has half a row of a tile: one exponential
// for a logit, whose 256 x 256 for a pair take half as long as 1024 terms of the product; below 512 terms they bound it.
template <int MODE, typename T, int BN, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1) products_kernel(const __grid_constant__ Products p) {
    constexpr int STAGES = kStages<BN, PAIR>, HALF = BN / 2, CTAS = PAIR ? 2 : 1;
    constexpr uint32_t STAGE = kStageBytes<BN, PAIR>;
    extern __shared__ uint8_t s_room[];
    const uint32_t room = (shared_address(s_room) + 1023) & ~1023u, staging = room + STAGES * STAGE;
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
            barrier_init(taken + 8 * s, 8 * CTAS);
        }
        barrier_init(drained, 1);
        *s_gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    if (warp == 1) tmem_alloc<PAIR>(s_tmem, 2 * BN);
    tmem_before_sync();
    if (PAIR) cluster_sync(); // (both CTAs' barriers are there)
    __syncthreads();
    tmem_after_sync();
    wait_for_previous();
    let_next_begin();
    const Head &h = p.head;
    const uint32_t tmem = *(volatile uint32_t *)(s_bias + 257);
    const int rows = rows_counted(h), rank = blockIdx.x % CTAS, unit = blockIdx.x / CTAS;
    const uint32_t first_full = PAIR ? there(full, 0) : full, first_taken = PAIR ? there(taken, 0) : taken;
    auto copy = [&](uint32_t to, const CUtensorMap *map, int x, int y, uint32_t bar) {
        if (PAIR)
            copy_box_of_pair(to, map, x, y, bar);
        else
            copy_box(to, map, x, y, bar);
    };
    Tile tile;
    Waiter waiter(s_gave_up);
    const bool &fine = waiter.fine;
    if (warp == 0) {
        if (lane == 0) {
            uint32_t n = 0; // stages filled so far
            for (Walk<MODE> walk(p, rows, unit); fine && walk.next(p, rows, tile);) {
                const Product &w = p.of[tile.product];
                for (int k = tile.from; k < tile.to; k++, n++) {
                    const uint32_t s = n % STAGES, at = room + s * STAGE, bar = first_full + 8 * s;
                    const int row = tile.row * (128 * CTAS) + rank * 128, column = tile.column * BN + rank * (BN / CTAS); // of this CTA
                    if (n >= STAGES && !barrier_wait(waiter, empty + 8 * s, (n / STAGES - 1) & 1)) break;
                    if (rank == 0) barrier_expect(full + 8 * s, CTAS * STAGE);
                    if (MODE == kProducts) {
                        if (w.a_along_sum) {
                            copy(at, &w.a, row, k * kSum, bar);
                            copy(at + kRowsBytes / 2, &w.a, row + 64, k * kSum, bar);
                        } else {
                            copy(at, &w.a, k * kSum, row, bar);
                        }
#pragma unroll
                        for (int j = 0; j < BN / CTAS / 64; j++) copy(at + kRowsBytes + j * (kSum * 128), &w.b, column + 64 * j, w.b_first + k * kSum, bar);
                    } else {
                        copy(at, &w.a, k * kSum, row, bar);
                        copy(at + kRowsBytes, &w.b, k * kSum, w.b_first + column, bar);
                    }
                }
            }
            if (PAIR) // nothing arrives behind the pair's end: no word that a stage is free, from the other CTA
                for (uint32_t k = n < STAGES ? 0 : n - STAGES; k < n; k++) barrier_wait(waiter, empty + 8 * (k % STAGES), k / STAGES & 1);
            if (rank == 0 && !(PAIR && fine)) // nor a copy (or the other CTA's), which nobody has waited for where the others have given up
                for (uint32_t k = n < STAGES ? 0 : n - STAGES; k < n; k++) {
                    volatile int mine = 0;
                    Waiter patient(&mine);
                    barrier_wait(patient, full + 8 * (k % STAGES), k / STAGES & 1);
                }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            uint32_t n = 0, m = 0; // stages and tiles multiplied so far
            for (Walk<MODE> walk(p, rows, unit); fine && walk.next(p, rows, tile);) {
                const bool a_along_sum = MODE == kProducts && p.of[tile.product].a_along_sum;
                const uint32_t kind = product_kind(sizeof(T) == 2 && kHeld<T> == 1.0f, 128 * CTAS, BN, a_along_sum, MODE == kProducts), half = m & 1;
                if (m >= 2 && !barrier_wait(waiter, taken + 8 * half, (m / 2 - 1) & 1)) break;
                tmem_after_sync();
                for (int k = tile.from; k < tile.to; k++, n++) {
                    const uint32_t s = n % STAGES, at = room + s * STAGE;
                    if (!barrier_wait(waiter, full + 8 * s, n / STAGES & 1)) break;
                    tmem_after_sync();
                    const uint64_t a = operand(at, kSum * 128), b = operand(at + kRowsBytes, kSum * 128);
#pragma unroll
                    for (int i = 0; i < kSum / 16; i++) // 16 terms: 32 bytes along a box's rows, or 16 of them
                        multiply<PAIR>(tmem + half * BN, a + i * (a_along_sum ? 128 : 2), b + i * (MODE == kProducts ? 128 : 2), kind, k > tile.from || i > 0);
                    when_multiplied<PAIR>(empty + 8 * s);
                }
                if (!fine) break;
                when_multiplied<PAIR>(done + 8 * half);
                m++;
            }
            if (!fine) {
                volatile int mine = 0;
                Waiter patient(&mine);
                when_multiplied<PAIR>(drained);
                barrier_wait(patient, drained, 0);
            }
        }
        __syncwarp();
    } else {
        const int quarter = warp & 3, side = (warp - 2) >> 2; // 32 rows, half of the columns
        const uint32_t mine = staging + (warp - 2) * 4096, my_row = mine + lane * 128;
        const uint32_t from = tmem + ((uint32_t)quarter << 21) + side * HALF;
        const float k_all = MODE == kProducts ? gradient_scale<T>(h) : 0.0f;
        uint32_t m = 0;
        for (Walk<MODE> walk(p, rows, unit); walk.next(p, rows, tile);) {
            const Product &w = p.of[tile.product];
            const uint32_t half = m & 1, at = from + half * BN;
            const int row_tile = tile.row * CTAS + rank, row = row_tile * 128 + quarter * 32 + lane, column = tile.column * BN + side * HALF; // (of the lane; the first)
            if (MODE != kProducts) { // the columns' bias; classes that there are not have a logit of -inf
                asm volatile("bar.sync 1, 256;" ::: "memory");
                if (threadIdx.x - 64 < BN) {
                    const int c = h.first + tile.column * BN + (int)threadIdx.x - 64;
                    s_bias[threadIdx.x - 64] = c >= h.a.classes ? -INFINITY : h.a.bias ? to_float(static_cast<const T *>(h.a.bias)[c]) : 0.0f;
                }
                asm volatile("bar.sync 1, 256;" ::: "memory");
            }
            barrier_wait(waiter, done + 8 * half, m / 2 & 1);
            waiter.fine = __all_sync(0xffffffffu, fine); // (and stays so for all tiles that are left)
            tmem_after_sync();
            m++;
            auto give_back = [&] { // behind the last load of the tile (one that has given up would be ahead of the others, and their half multiplied over)
                tmem_before_sync();
                __syncwarp();
                if (lane != 0 || !fine) return;
                if (PAIR)
                    barrier_arrive_there(first_taken + 8 * half);
                else
                    barrier_arrive(taken + 8 * half);
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
                    tmem_wait(raw);
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
                    if (apart) away += h.share * (float)min(c, max(left, 0)) * fmaxf(top - most, kLowest);
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
                        for (int j = 0; j < 16; j++) all += h.share * (c + 2 * j < left ? z[j].lo() : 0.0f) + h.share * (c + 2 * j + 1 < left ? z[j].hi() : 0.0f);
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
                            const float most = *h.most, mine = h.a.upstream[orig];
                            held *= !(fabsf(mine) < INFINITY) ? NAN : most == 0.0f ? 0.0f : mine / most;
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
                // (what is there is no number, perhaps)
                const bool blank = MODE == kGradient ? row >= rows : w.counted == kSumCounted && rows == 0;
                const bool part = MODE == kProducts && !tile.whole;
                const float times_it = part || (MODE == kProducts && w.leaves != kWritten) ? 1.0f : factor;
                const Two minus(-row_top, -row_top), log2e(kLog2e, kLog2e), times(times_it, times_it), less(-flat, -flat);
                // a part's place: the run's first, or its last
                const int row0 = (part ? 2 * (int)blockIdx.x + (tile.from == 0) : row_tile) * 128 + quarter * 32;
                const int x0 = part ? side * HALF : column, x_last = part ? BN : MODE == kGradient ? h.columns : (int)h.a.width;
                // 32 columns from c on
                auto values = [&](Two(&v)[16], const uint32_t(&raw)[32], int c) {
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        Two a(__uint_as_float(raw[j]), __uint_as_float(raw[j + 1])), b(__uint_as_float(raw[j + 2]), __uint_as_float(raw[j + 3]));
                        if constexpr (MODE == kGradient) {
                            const float4 bias = bias4[(c + j) / 4];
                            a = mul_rn(add_rn(add_rn(a, Two(bias.x, bias.y)), minus), log2e);
                            b = mul_rn(add_rn(add_rn(b, Two(bias.z, bias.w)), minus), log2e);
                            a = fma_rn(Two(exp2_of(a.lo()), exp2_of(a.hi())), times, less);
                            b = fma_rn(Two(exp2_of(b.lo()), exp2_of(b.hi())), times, less);
                        } else {
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
                auto leave = [&](int c) {
                    shared_to_copies();
                    __syncwarp();
                    if (lane == 0 && x0 + c < x_last && (part || row0 < w.c_last)) {
                        if (part)
                            store_box(&p.part, x0 + c, row0, mine);
                        else if (MODE == kProducts && w.leaves == kAdded32)
                            add_box(&w.c, x0 + c, row0, mine);
                        else
                            store_box(&w.c, x0 + c, row0, mine);
                        boxes_commit();
                    }
                };
                if (MODE == kGradient || (w.leaves == kWritten && !part)) {
#pragma unroll 1
                    for (int c = 0; c < HALF; c += 64) {
                        uint32_t raw[2][32], out[32];
                        Two v[2][16];
                        tmem_load(raw[0], at + c);
                        tmem_load(raw[1], at + c + 32);
                        tmem_wait(raw[0]);
                        tmem_wait(raw[1]);
                        if (c + 64 >= HALF) give_back();
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            values(v[i], raw[i], c + 32 * i);
#pragma unroll
                            for (int j = 0; j < 16; j++) out[16 * i + j] = two_of<T>(v[i][j].lo(), v[i][j].hi());
                        }
                        room_free(); // (the last box has been read meanwhile)
#pragma unroll
                        for (int j = 0; j < 8; j++) piece(j, make_uint4(out[4 * j], out[4 * j + 1], out[4 * j + 2], out[4 * j + 3]));
                        if constexpr (MODE == kGradient) {
#pragma unroll
                            for (int k = 0; k < 2; k++) {
                                const int l = label[k] - c;
                                if (label[k] < 0 || l < 0 || l >= 64) continue;
                                const uint32_t two = two_of<T>(fine ? written[k] : NAN, 0.0f);
                                asm volatile("st.shared.b16 [%0], %1;" ::"r"(my_row + ((l / 8 ^ (lane & 7)) << 4) + l % 8 * 2), "h"((uint16_t)two) : "memory");
                            }
                        }
                        leave(c);
                        if constexpr (MODE == kGradient) {
                            if (h.bias_parts) { // sums of these 32 rows, before they are rounded
#pragma unroll
                                for (int k = 0; k < 2; k++) {
                                    const int l = label[k] < 0 ? -1 : label[k] - c;
                                    const float one = fine ? written[k] : NAN;
                                    if (__any_sync(0xffffffffu, l >= 0 && l < 64)) {
#pragma unroll
                                        for (int j = 0; j < 32; j++)
                                            v[j / 16][j % 16] = Two(l == 2 * j ? one : v[j / 16][j % 16].lo(), l == 2 * j + 1 ? one : v[j / 16][j % 16].hi());
                                    }
                                }
                                float sum[2];
                                sum_rows(v, sum);
                                float *to = h.bias_parts + (long long)(row_tile * 4 + quarter) * h.chunk + column + c + lane;
#pragma unroll
                                for (int i = 0; i < 2; i++)
                                    if (column + c + 32 * i + lane < h.chunk) to[32 * i] = sum[i];
                            }
                        }
                    }
                } else {
#pragma unroll 1
                    for (int c = 0; c < HALF; c += 32) {
                        uint32_t raw[32];
                        tmem_load(raw, at + c);
                        tmem_wait(raw);
                        if (c + 32 >= HALF) give_back();
                        Two v[16];
                        values(v, raw, c);
                        room_free();
#pragma unroll
                        for (int j = 0; j < 8; j++)
                            piece(j, make_uint4(__float_as_uint(v[2 * j].lo()), __float_as_uint(v[2 * j].hi()), __float_as_uint(v[2 * j + 1].lo()), __float_as_uint(v[2 * j + 1].hi())));
                        leave(c);
                    }
                }
            }
        }
        if (MODE != kStatistics && lane == 0) boxes_written();
        __syncwarp();
    }
    tmem_before_sync();
    __syncthreads();
    if (PAIR) cluster_sync(); // (nothing of the other CTA's arrives here any more)
    tmem_after_sync();
    if (warp == 1) tmem_free<PAIR>(tmem, 2 * BN);
}

// Rows' statistics joined over the classes: 32 rows per CTA, whose warps take the parts in turn: of 8192 x 171 16 MB, 9 us.
__global__ void __launch_bounds__(1024) join_kernel(const __grid_constant__ Head h) {
    __shared__ float s_top[32][33], s_sum[32][33], s_away[32][33], s_row[3][32];
    wait_for_previous();
    let_next_begin();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, rows = rows_counted(h);
    if (blockIdx.x * 32 >= rows) return;
    const bool apart = h.a.smoothing > 0.0f;
    float top = kLowest, sum = 0.0f, away = 0.0f, mass = 0.0f; // (mass: what the classes seen have of the target by smoothing)
    auto add = [&](float t, float s, float d, float there) {
        const float most = fmaxf(top, t);
        sum = sum * exp_of(top - most) + s * exp_of(t - most);
        if (apart) {
            away += mass * fmaxf(top - most, kLowest) + d + there * fmaxf(t - most, kLowest);
            mass += there;
        }
        top = most;
    };
    auto there_of = [&](int k) { return h.share * (float)max(0, min(h.part_columns, (int)h.a.classes - k * h.part_columns)); };
    {
        const int row = blockIdx.x * 32 + lane;
#pragma unroll 4
        for (int k = warp; k < h.part_count; k += warps) {
            const long long at = (long long)k * h.rows_pad + row;
            const float2 one = h.parts[at];
            add(one.x, one.x != one.x ? NAN : one.y, apart ? h.parts_apart[at] : 0.0f, there_of(k));
        }
    }
    s_top[warp][lane] = top, s_sum[warp][lane] = sum, s_away[warp][lane] = away;
    __syncthreads();
    // now a warp has a row at a time, and a lane what a warp had of it
    for (int r = warp; r < 32; r += warps) {
        const float mine = lane < warps ? s_top[lane][r] : kLowest, most = warp_max(mine);
        const float whole = warp_sum(lane < warps ? s_sum[lane][r] * exp_of(mine - most) : 0.0f);
        float apart_all = 0.0f;
        if (apart) {
            float seen = 0.0f;
            if (lane < warps)
                for (int k = lane; k < h.part_count; k += warps) seen += there_of(k);
            apart_all = warp_sum(lane < warps ? s_away[lane][r] + seen * fmaxf(mine - most, kLowest) : 0.0f);
        }
        if (lane == 0) s_row[0][r] = most, s_row[1][r] = whole, s_row[2][r] = apart_all;
    }
    __syncthreads();
    const int row = blockIdx.x * 32 + lane;
    if (warp || row >= rows) return;
    const float most = s_row[0][lane], whole = s_row[1][lane];
    const long long orig = h.map ? h.map[row] : row;
    const Picks p = picks_of(h.a, orig);
    float4 *stats = reinterpret_cast<float4 *>(h.a.stats) + orig;
    float loss = NAN, over = NAN;
    if (!p.bad) {
        const float picked[2] = {stats->z, stats->w};
        float dot = p.flat > 0.0f ? s_row[2][lane] : 0.0f;
        for (int k = 0; k < 2; k++)
            if (p.weight[k] != 0.0f) dot += p.weight[k] * (picked[k] - most);
        loss = whole == 0.0f ? 0.0f : p.total * logf(whole) - dot;
        over = whole == 0.0f ? 0.0f : 1.0f / whole;
    }
    h.a.row_loss[orig] = loss;
    stats->x = most;
    stats->y = over;
}

// Which rows count, in their order: the place of each, or -1; a row for each place.  Rows that do not count get a loss of 0.  One cluster of eight CTAs, which tell one
// another how many they have: 50176 rows 9 us, 49 by one CTA.
constexpr int kPlacesCtas = 8;
__global__ void __launch_bounds__(1024) places_kernel(const __grid_constant__ ffcvb_linear_cross_entropy_args a, int *map, int *place, float *counted) {
    __shared__ int s_count[32], s_before[kPlacesCtas];
    wait_for_previous();
    let_next_begin();
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); // (this one has begun)
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t *labels = static_cast<const int64_t *>(a.target);
    // a warp has a run of rows, 32 at a time, eight loads ahead
    const int run = (int)((a.rows + kPlacesCtas * 1024 - 1) / (kPlacesCtas * 1024)) * 32, first = (blockIdx.x * 32 + warp) * run, last = min(first + run, (int)a.rows);
    auto counting = [&](int r0) {
        int64_t label[8];
#pragma unroll
        for (int i = 0; i < 8; i++) label[i] = r0 + 32 * i + lane < last ? labels[(r0 + 32 * i + lane) * a.target_stride] : a.ignore_index;
        uint32_t bits = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) bits |= (label[i] != a.ignore_index ? 1u : 0u) << i;
        return bits;
    };
    int n = 0;
    for (int r0 = first; r0 < last; r0 += 256) n += __popc(counting(r0));
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) s_count[warp] = n;
    __syncthreads();
    int before = __reduce_add_sync(0xffffffffu, lane < warp ? s_count[lane] : 0);
    const int whole = __reduce_add_sync(0xffffffffu, s_count[lane]);
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); // all have begun
    if (threadIdx.x < kPlacesCtas) {
        uint32_t there;
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(shared_address(s_before + blockIdx.x)), "r"(threadIdx.x));
        asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(there), "r"(whole) : "memory");
    }
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    for (int k = 0; k < (int)blockIdx.x; k++) before += s_before[k];
    if (blockIdx.x == kPlacesCtas - 1 && warp == 31 && lane == 0) *counted = (float)(before + n);
    for (int r0 = first; r0 < last; r0 += 256) {
        const uint32_t bits = counting(r0);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int r = r0 + 32 * i + lane;
            const bool counts = bits >> i & 1;
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
    }
}

// Rows of `width` values of 16 bits in places that the copies can begin at; rows behind those that count, up to the next 128, and columns behind
// the last one are 0.  A copy: 50176 x 768 11 us where 40 % of the rows count.
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

// The largest size of the upstream gradients of rows that count (place: as of places_kernel, or NULL).  One that is no number or has no end is left out: it is
// its own row's, whose G is NaN, and not the scale of the others.
__global__ void __launch_bounds__(1024) most_kernel(const float *__restrict__ upstream, const int *__restrict__ place, long long rows, float *most) {
    __shared__ float s_most[32];
    wait_for_previous();
    let_next_begin();
    float m = 0.0f;
    for (long long i = threadIdx.x; i < rows; i += 1024) {
        const float v = fabsf(upstream[i]);
        if (v < INFINITY && (!place || place[i] >= 0)) m = fmaxf(m, v);
    }
    m = warp_max(m);
    if ((threadIdx.x & 31) == 0) s_most[threadIdx.x >> 5] = m;
    __syncthreads();
    if (threadIdx.x < 32) {
        m = warp_max(s_most[threadIdx.x]);
        if (threadIdx.x == 0) *most = m;
    }
}

// Gradients from sums in 32 bits, or of rows that count from 16 bits: out[r] = from[place of r]; rows without a place are 0.  Bound by HBM: 8192 x 1024 sums 9 us, 50176 x 768
// from 40 % as many sums 22.
template <typename T, typename From>
__global__ void __launch_bounds__(256) settle_kernel(const __grid_constant__ Head h, const From *__restrict__ sums, int pad, const int *place, T *__restrict__ out, int rows, int width) {
    wait_for_previous();
    let_next_begin();
    const float k = sizeof(From) == 4 ? gradient_scale<T>(h) : 1.0f;
    const int packs = (width + 7) / 8;
    const bool wide = width % 8 == 0;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < (long long)rows * packs; i += (long long)gridDim.x * 256) {
        const int r = (int)(i / packs), c = (int)(i - (long long)r * packs) * 8, from = place ? place[r] : r;
        float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
        if (from >= 0) {
            const From *at = sums + (long long)from * pad + c;
            constexpr int N = kWide<From>;
#pragma unroll
            for (int j = 0; j < 8; j += N) {
                Pack<From, N> pack;
                float f[N];
                pack.load(at + j);
                pack.get(f);
#pragma unroll
                for (int l = 0; l < N; l++) v[j + l] = f[l] * k;
            }
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

// What is left to do behind a chunk's products: tiles that several CTAs have parts of, added up in their order; and the bias' gradient.  The first CTAs have
// 32 classes each, whose sums over 32 rows they add up; the others 32 rows each of the tile that a run begins in the middle of (the first such run of a tile).
// 7 to 16 us, for which all runs end at once: whole tiles dealt out to 148 CTAs leave up to half of them idle in the last turn (8192 x 21841 x 1024: 1720 us and 1348).
template <typename T, int BN>
__global__ void __launch_bounds__(256) finish_kernel(const __grid_constant__ Products p) {
    __shared__ float s_sum[8][32];
    wait_for_previous();
    let_next_begin();
    const Head &h = p.head;
    const int rows = rows_counted(h), pieces = p.high / 32, biases = h.bias_parts ? (h.columns + 31) / 32 : 0;
    if ((int)blockIdx.x < biases) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = (int)blockIdx.x * 32 + lane, parts = (rows + 127) / 128 * 4;
        float sum = 0.0f;
        if (c < h.columns) {
#pragma unroll 16
            for (int k = warp; k < parts; k += 8) sum += h.bias_parts[(long long)k * h.chunk + c];
        }
        s_sum[warp][lane] = sum;
        __syncthreads();
        if (warp || c >= h.columns) return;
        for (int k = 1; k < 8; k++) sum += s_sum[k][lane];
        static_cast<T *>(h.a.grad_bias)[h.first + c] = from_float<T>(sum * gradient_scale<T>(h));
        return;
    }
    const Runs runs(p, rows);
    const int n = (int)blockIdx.x - biases, unit = n / pieces, piece = n - unit * pieces, place = runs.place(unit), lane = runs.lane(unit);
    if (place == 0 || place >= runs.units) return;
    const int begin = runs.begin(place);
    const Tile tile = tile_of(p, runs, lane, begin, rows);
    if (tile.from == 0 || begin - runs.begin(place - 1) < tile.from) return; // (a run's own tile; one that an earlier run has begun in the middle of)
    int last = place; // the last run with a part
    while (last + 1 < runs.units && runs.begin(last + 1) - begin < tile.to - tile.from) last++;
    const Product &w = p.of[tile.product];
    const float k = w.leaves == kWritten ? gradient_scale<T>(h) : 1.0f;
    const bool blank = w.counted == kSumCounted && rows == 0;
    for (int i = threadIdx.x; i < 32 * BN / 8; i += 256) {
        const int r = piece % 4 * 32 + i / (BN / 8), c = i % (BN / 8) * 8, row = tile.row * p.high + piece * 32 + i / (BN / 8), column = tile.column * BN + c;
        if (row >= w.c_last || column >= h.a.width) continue;
        float v[8];
        auto take = [&](int unit, int end, bool first) { // (of a pair's CTA)
            const int part = 2 * (unit * (p.high / 128) + piece / 4) + end;
            const float *at = p.parts + ((long long)part * 128 + r) * BN + c;
#pragma unroll
            for (int j = 0; j < 8; j += 4) {
                const float4 f = *reinterpret_cast<const float4 *>(at + j);
                v[j] = first ? f.x : v[j] + f.x;
                v[j + 1] = first ? f.y : v[j + 1] + f.y;
                v[j + 2] = first ? f.z : v[j + 2] + f.z;
                v[j + 3] = first ? f.w : v[j + 3] + f.w;
            }
        };
        take(unit - runs.lanes, 1, true);
#pragma unroll 4
        for (int other = place; other <= last; other++) take(unit + (other - place) * runs.lanes, 0, false);
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = blank ? 0.0f : v[j] * k;
        if (w.leaves == kWritten) {
            Pack<T, 8> pack;
            pack.set(v);
            pack.store(static_cast<T *>(w.out) + row * w.out_stride + column);
            continue;
        }
        float *to = static_cast<float *>(w.out) + row * w.out_stride + column;
#pragma unroll
        for (int j = 0; j < 8; j += 4) {
            float4 out = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
            if (w.leaves == kAdded32) {
                const float4 was = *reinterpret_cast<const float4 *>(to + j);
                out.x += was.x, out.y += was.y, out.z += was.z, out.w += was.w;
            }
            *reinterpret_cast<float4 *>(to + j) = out;
        }
    }
}

// ---- the host's part -------------------------------------------------------------------------------------------------

inline int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// What a call does, and where in the workspace (offsets in bytes).
struct Plan {
    int64_t rows_pad, width_pad, chunk, chunks;  // (classes at once)
    bool counted, lay_hidden, lay_weight, grads, hidden_grad, weight_grad, bias_grad;
    int stat_columns, sum_columns;               // BN
    bool hidden_direct, weight_direct;           // products leave as they are to be
    bool pairs;                                  // of CTAs
    int64_t map, place, count, most, hidden, weight, parts, apart, grad, hidden_sums, hidden_rows, weight_sums, bias_parts, tile_parts, bytes;
};

// G's bytes at most, or those of 256 classes of all rows: so many classes at once that the sum over classes of dx's few tiles is long and few parts are joined.  (8192 x 21841 x 1024, 358 MB in two chunks: 1038 us,
// 1080 with 128 MB, 1184 with 64, 1192 with 512, which is one chunk; 50176 x 8192 x 768, 822 MB: 2374, 2736, 2866 and 2522.)
constexpr int64_t kMostGradient = 256ll << 20;

bool aligned(const void *p, int64_t stride) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride % 8 == 0; }

// Columns of the logits' tiles: 256, but 128 where single CTAs would leave more than every other SM without a tile. Microseconds with 256 and with 128 columns: 4096 x
// 1000 x 768 55 and 60, 16384 x 200 x 768 66 and 70, 128 x 21841 x 1024 82 and 89; below the bound 64 x 1000 x 384 35 and 33, 64 x 100 x 128 27 and 24.
int columns_of(const Plan &p, int64_t classes) { return p.pairs || p.rows_pad / 128 * ((classes + 255) / 256) >= kSms / 2 ? 256 : 128; }

Plan plan_of(const ffcvb_linear_cross_entropy_args &a) {
    Plan p{};
    // Pairs where there are rows for the second CTA and a tile of 256 x 256 logits for every SM: 1021 x 21841 x 768 takes 132 us, 166 by single CTAs; 512 x 10000 x
    // 1024 (80 tiles) takes 79 either way, 1000 x 5000 x 512 (80 tiles) 55 by single CTAs and 64 by pairs, 128 x 21841 x 1024 (86 tiles, one of the two CTAs idle) 71
    // and 108.
    p.pairs = a.rows > 128 && (a.rows + 255) / 256 * ((a.classes + 255) / 256) >= kSms;
    p.rows_pad = up(a.rows, p.pairs ? 256 : 128);
    p.width_pad = up(a.width, 8);
    p.counted = a.has_ignore && a.target_kind == FFCVB_TARGET_LABELS;
    p.lay_hidden = p.counted || !aligned(a.hidden, a.hidden_stride);
    p.lay_weight = !aligned(a.weight, a.weight_stride);
    p.hidden_grad = a.grad_hidden, p.weight_grad = a.grad_weight, p.bias_grad = a.grad_bias;
    p.grads = p.hidden_grad || p.weight_grad || p.bias_grad;
    p.stat_columns = columns_of(p, a.classes);
    p.chunks = (a.classes * p.rows_pad * 2 + kMostGradient - 1) / kMostGradient;
    p.chunk = up((a.classes + p.chunks - 1) / p.chunks, 256);
    p.chunks = (a.classes + p.chunk - 1) / p.chunk;
    p.sum_columns = p.pairs ? 256 : 128; // (single CTAs with 128 and with 256 columns: 64 x 1000 x 384 29 us and 33, 4096 x 100 x 384 41 and 49, 128 x 21841 x 1024 77 and 89)
    p.hidden_direct = p.chunks == 1 && (p.counted || a.width % 8 == 0);
    p.weight_direct = a.width % 8 == 0;
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
    p.hidden_sums = take(p.hidden_grad && !p.hidden_direct, p.rows_pad * wide * 4);
    p.hidden_rows = take(p.hidden_grad && p.hidden_direct && p.counted, p.rows_pad * p.width_pad * 2);
    p.weight_sums = take(p.weight_grad && !p.weight_direct, p.chunk * wide * 4);
    p.tile_parts = take(p.hidden_grad || p.weight_grad, 2ll * kSms * 128 * p.sum_columns * 4);
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
    if (((reinterpret_cast<uintptr_t>(a.grad_hidden) | reinterpret_cast<uintptr_t>(a.grad_weight) | reinterpret_cast<uintptr_t>(a.stats)) & 15) != 0) return "gradients and stats begin on 16 bytes";
    return nullptr;
}

template <int MODE, typename T, int BN, bool PAIR> bool launch_products(Products &p, int64_t tiles, cudaStream_t stream) {
    auto *kernel = products_kernel<MODE, T, BN, PAIR>;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kRoom<BN, PAIR>) != cudaSuccess) return false;
    constexpr int CTAS = PAIR ? 2 : 1;
    p.units = (int)std::min<int64_t>(tiles, kSms / CTAS);
    cudaLaunchConfig_t how{};
    cudaLaunchAttribute with[2] = {};
    with[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    with[0].val.programmaticStreamSerializationAllowed = 1;
    with[1].id = cudaLaunchAttributeClusterDimension;
    with[1].val.clusterDim.x = CTAS;
    with[1].val.clusterDim.y = with[1].val.clusterDim.z = 1;
    how.gridDim = dim3((unsigned)(p.units * CTAS));
    how.blockDim = dim3(kThreads);
    how.dynamicSmemBytes = kRoom<BN, PAIR>;
    how.stream = stream;
    how.attrs = with;
    how.numAttrs = PAIR ? 2 : 1;
    return cudaLaunchKernelEx(&how, kernel, p) == cudaSuccess;
}
template <int MODE, typename T> bool launch_products(int columns, bool pairs, Products &p, int64_t tiles, cudaStream_t stream) {
    if (pairs) return launch_products<MODE, T, 256, true>(p, tiles, stream);
    return columns == 256 ? launch_products<MODE, T, 256, false>(p, tiles, stream) : launch_products<MODE, T, 128, false>(p, tiles, stream);
}

template <typename T> int run(const ffcvb_linear_cross_entropy_args &a, uint8_t *room, cudaStream_t st) {
    const Plan p = plan_of(a);
    const int type = a.type;
    const int high = p.pairs ? 256 : 128;
    const int64_t row_tiles = p.rows_pad / high;
    auto at = [&](int64_t offset) { return static_cast<void *>(room + offset); };
    Products g{};
    g.high = high;
    Head &h = g.head;
    h.a = a;
    h.share = a.smoothing / (float)a.classes;
    h.rows_pad = (int)p.rows_pad;
    h.map = p.counted ? static_cast<int *>(at(p.map)) : nullptr;
    h.place = p.counted ? static_cast<int *>(at(p.place)) : nullptr;
    h.counted = p.counted ? static_cast<float *>(at(p.count)) : nullptr;
    h.most = static_cast<float *>(at(p.most));
    h.parts = static_cast<float2 *>(at(p.parts));
    h.parts_apart = static_cast<float *>(at(p.apart));
    h.part_columns = p.stat_columns / 2;
    h.part_count = (int)(up(a.classes, p.stat_columns) / h.part_columns);
    if (p.counted) {
        cudaLaunchConfig_t how{};
        cudaLaunchAttribute with[2] = {};
        with[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        with[0].val.programmaticStreamSerializationAllowed = 1;
        with[1].id = cudaLaunchAttributeClusterDimension;
        with[1].val.clusterDim.x = kPlacesCtas;
        with[1].val.clusterDim.y = with[1].val.clusterDim.z = 1;
        how.gridDim = dim3(kPlacesCtas);
        how.blockDim = dim3(1024);
        how.stream = st;
        how.attrs = with;
        how.numAttrs = 2;
        cudaLaunchKernelEx(&how, places_kernel, a, static_cast<int *>(at(p.map)), static_cast<int *>(at(p.place)), static_cast<float *>(at(p.count)));
    }
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
    Product of_logits{};
    int mapped_columns = 0; // (the maps, 0.3 us each, are made once)
    auto logits = [&](int columns, int64_t first, int64_t count) {
        if (mapped_columns != columns) {
            mapped &= matrix_map(&of_logits.a, type, hidden, hidden_rows, a.width, hidden_stride, 128);
            mapped &= matrix_map(&of_logits.b, type, weight, a.classes, a.width, weight_stride, p.pairs ? columns / 2 : columns);
            mapped_columns = columns;
        }
        Product &w = g.of[0];
        w = of_logits;
        w.row_tiles = (int)row_tiles;
        w.column_tiles = (int)((count + columns - 1) / columns);
        w.sum_blocks = sum_blocks;
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
        fine &= launch_products<kStatistics, T>(p.stat_columns, p.pairs, g, tiles, st);
        // (32 warps, or eight where there are two CTAs for every SM: 1021 x 21841 x 768 130 us and 136, 50176 x 1000 x 256 195 and 187)
        launch_early(join_kernel, (unsigned)(p.rows_pad / 32), p.rows_pad / 32 >= 2 * kSms ? 256 : 1024, 0, st, h);
        if (a.loss) launch_mean(a.row_loss, a.rows, h.counted, a.mean, a.loss, st);
    }
    if (!p.grads) return fine ? launched("ffcvb_linear_cross_entropy") : training_fail(FFCVB_E_CUDA, "ffcvb_linear_cross_entropy: %s", cudaGetErrorString(cudaGetLastError()));
    if (a.upstream && a.upstream_per_row) launch_early(most_kernel, 1, 1024, 0, st, a.upstream, h.place, a.rows, static_cast<float *>(at(p.most)));
    const int64_t wide = up(a.width, 32);
    auto ctas_for = [&](int64_t rows) { return (unsigned)std::min<int64_t>((rows * ((a.width + 7) / 8) + 255) / 256, kSms * 8); };
    for (int64_t chunk = 0; chunk < p.chunks; chunk++) {
        const int64_t first = chunk * p.chunk, count = std::min(p.chunk, a.classes - first);
        const int columns = columns_of(p, count);
        int64_t tiles = logits(columns, first, count);
        mapped &= matrix_map(&g.of[0].c, type, at(p.grad), p.counted ? p.rows_pad : a.rows, count, p.chunk, 32);
        g.of[0].c_last = (int)(p.counted ? p.rows_pad : a.rows);
        h.bias_parts = p.bias_grad ? static_cast<float *>(at(p.bias_parts)) : nullptr;
        h.chunk = (int)p.chunk;
        if (!mapped) break;
        fine &= launch_products<kGradient, T>(columns, p.pairs, g, tiles, st);
        const int column_tiles = (int)((a.width + p.sum_columns - 1) / p.sum_columns);
        g.count = 0;
        g.lanes = column_tiles <= 16 ? column_tiles : 1; // (few CTAs are left without one)
        // C: in what it is to be, in rows that count, or in 32 bits
        auto leaves_as = [&](Product &w, int how, void *out, int64_t rows, int64_t stride) {
            w.leaves = how;
            w.out = out;
            w.out_stride = stride;
            w.c_last = (int)rows;
            w.column_tiles = column_tiles;
            mapped &= matrix_map(&w.c, how == kWritten ? type : FFCVB_TYPE_F32, out, rows, how == kWritten ? a.width : wide, stride, 32);
        };
        if (p.hidden_grad) {
            Product &w = g.of[g.count++];
            mapped &= matrix_map(&w.a, type, at(p.grad), p.counted ? p.rows_pad : a.rows, count, p.chunk, 128);
            mapped &= matrix_map(&w.b, type, weight, a.classes, a.width, weight_stride, kSum);
            if (!p.hidden_direct)
                leaves_as(w, chunk ? kAdded32 : kWritten32, at(p.hidden_sums), p.rows_pad, wide);
            else if (p.counted)
                leaves_as(w, kWritten, at(p.hidden_rows), p.rows_pad, p.width_pad);
            else
                leaves_as(w, kWritten, a.grad_hidden, a.rows, a.width);
            w.row_tiles = (int)row_tiles;
            w.sum_blocks = (int)((count + kSum - 1) / kSum);
            w.a_along_sum = 0;
            w.counted = p.counted ? kRowsCounted : kFixed;
            w.b_first = (int)first;
        }
        if (p.weight_grad) {
            Product &w = g.of[g.count++];
            mapped &= matrix_map(&w.a, type, at(p.grad), p.counted ? p.rows_pad : a.rows, count, p.chunk, kSum);
            mapped &= matrix_map(&w.b, type, hidden, hidden_rows, a.width, hidden_stride, kSum);
            if (p.weight_direct)
                leaves_as(w, kWritten, static_cast<T *>(a.grad_weight) + first * a.width, count, a.width);
            else
                leaves_as(w, kWritten32, at(p.weight_sums), p.chunk, wide);
            w.row_tiles = (int)((count + high - 1) / high);
            w.sum_blocks = (int)((a.rows + kSum - 1) / kSum);
            w.a_along_sum = 1;
            w.counted = p.counted ? kSumCounted : kFixed;
            w.b_first = 0;
        }
        if (g.count) {
            g.parts = static_cast<float *>(at(p.tile_parts));
            mapped &= matrix_map(&g.part, FFCVB_TYPE_F32, at(p.tile_parts), 2 * kSms * 128, p.sum_columns, p.sum_columns, 32);
        }
        if (!mapped) break;
        if (g.count) fine &= launch_products<kProducts, T>(p.sum_columns, p.pairs, g, kSms, st);
        const unsigned finish = (unsigned)((g.count ? g.units * (high / 32) : 0) + (p.bias_grad ? (count + 31) / 32 : 0));
        if (finish) launch_early(p.sum_columns == 256 ? finish_kernel<T, 256> : finish_kernel<T, 128>, finish, 256, 0, st, g);
        if (p.weight_grad && !p.weight_direct)
            launch_early(settle_kernel<T, float>, ctas_for(count), 256, 0, st, h, static_cast<const float *>(at(p.weight_sums)), (int)wide, (const int *)nullptr,
                         static_cast<T *>(a.grad_weight) + first * a.width, (int)count, (int)a.width);
    }
    if (!mapped) return training_fail(FFCVB_E_CUDA, "ffcvb_linear_cross_entropy: no map of a matrix");
    if (p.hidden_grad && !p.hidden_direct)
        launch_early(settle_kernel<T, float>, ctas_for(a.rows), 256, 0, st, h, static_cast<const float *>(at(p.hidden_sums)), (int)wide, h.place, static_cast<T *>(a.grad_hidden),
                     (int)a.rows, (int)a.width);
    else if (p.hidden_grad && p.counted)
        launch_early(settle_kernel<T, T>, ctas_for(a.rows), 256, 0, st, h, static_cast<const T *>(at(p.hidden_rows)), (int)p.width_pad, h.place, static_cast<T *>(a.grad_hidden),
                     (int)a.rows, (int)a.width);
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
