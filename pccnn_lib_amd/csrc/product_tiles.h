// Products of the feed-forward operators (gated.hip, eight_bit.hip): tiles of rows in LDS, 32 x 32 blocks of results in
// registers.  The layouts are those of attention_tiles.h: a product C = A B has C's column in the lane and C's rows in the
// registers, an operand is sixteen bytes of one row.  Here the lane's side are points (rows of the result), the registers' side
// output channels, so a lane holds runs of four neighboring channels of one point.
//
// Operands are bf16 or 8-bit integers whose rows start at multiples of 16 bytes and have whole 16-byte units (zeros behind the
// last element); whatever is not like that is laid out so first (product_stage_kernel), f32 as three planes of bf16 terms, whose
// tiles lie in LDS together: a product of f32 operands is the sum of the six products of planes whose indices add up to at most 2,
// smallest first.  Where a product leaves f32 its terms' products are infinities of both signs, and an infinite operand's second
// term is infinite, its third NaN: f32 results that are not finite are formed again by the f32 matrix instructions (settle), a block
// of 32 x 32 at a time, and are then what f32 arithmetic gives.
#pragma once
#include "attention_tiles.h"

#include <algorithm>
#include <float.h>
#include <type_traits>

#ifdef __HIPCC__
typedef int pccnn_i32x4 __attribute__((ext_vector_type(4)));
typedef int pccnn_i32x16 __attribute__((ext_vector_type(16)));
typedef float pccnn_f32x4 __attribute__((ext_vector_type(4)));
#endif

// One operand: rows of 16-byte units.  In bytes: the distance of rows, of the next 128 bytes of a row (128 where the row lies in
// one piece), of the planes of terms (f32; else there is one).
struct ProductRows {
    const void *p;
    int64_t stride, rows, plane, step = 128;
};

// The tiles of a product in the order of their workgroups: those of a tile of rows one behind the other, runs of 2^run_log2 of them
// on one XCD, whose L2 then serves the rows.  Numbers come apart by shifts and a multiplication with 2^shift / tiles rounded up
// (exact below 2^31): the divisions themselves were a hundred instructions, as much as six results of a gelu.
struct ProductGrid {
    uint32_t blocks, tiles, magic;
    int shift, run_log2;
};
static inline ProductGrid product_grid(int64_t tiles_m, int64_t tiles_n)
{
    ProductGrid g = {(uint32_t)(tiles_m * tiles_n), (uint32_t)tiles_n, 0, 31, 0};
    while (((int64_t)1 << (g.shift - 31)) < tiles_n) ++g.shift;
    g.magic = (uint32_t)((((uint64_t)1 << g.shift) + tiles_n - 1) / tiles_n);
    // as many as a tile of rows has, 64 at most, and no more than leave every XCD one
    while (((int64_t)1 << g.run_log2) < tiles_n && g.run_log2 < 6 && ((uint64_t)PCCNN_XCDS << (g.run_log2 + 1)) <= g.blocks) ++g.run_log2;
    return g;
}
static inline uint32_t product_workgroups(const ProductGrid &g)
{
    const uint32_t super = (uint32_t)PCCNN_XCDS << g.run_log2;
    return (g.blocks + super - 1) / super * super;
}

#ifdef __HIPCC__
// The tile of workgroup `at`, in scalar registers; false: it has none.
__device__ __forceinline__ bool product_tile(const ProductGrid &g, uint32_t at, uint32_t &row_tile, uint32_t &col_tile)
{
    const uint32_t within = at & ((PCCNN_XCDS << g.run_log2) - 1);
    const uint32_t block = at - within + ((within % PCCNN_XCDS) << g.run_log2) + within / PCCNN_XCDS;
    if (block >= g.blocks) return false;
    row_tile = (uint32_t)(((uint64_t)block * g.magic) >> g.shift);
    col_tile = block - row_tile * g.tiles;
    return true;
}

// What operands are multiplied as: TERMS planes, UNIT elements to 16 bytes, UNITS units of a row in LDS at a time.  One plane takes
// whole lines of L2 (128 bytes); three planes, with six products to a unit, half of them.
struct ProductBf16 {
    typedef pccnn_f32x16 Acc;
    static constexpr int TERMS = 1, UNIT = 8, UNITS = 8;
    static __device__ __forceinline__ Acc mma(const pccnn_u32x4 (&a)[1], const pccnn_u32x4 (&b)[1], Acc c)
    {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(pccnn_bf16x8, a[0]),
                                                       __builtin_bit_cast(pccnn_bf16x8, b[0]), c, 0, 0, 0);
    }
};
struct ProductF32 {
    typedef pccnn_f32x16 Acc;
    static constexpr int TERMS = 3, UNIT = 8, UNITS = 4;
    static __device__ __forceinline__ Acc mma(const pccnn_u32x4 (&a)[3], const pccnn_u32x4 (&b)[3], Acc c)
    {
        auto one = [&](int i, int j) {
            c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(pccnn_bf16x8, a[i]),
                                                        __builtin_bit_cast(pccnn_bf16x8, b[j]), c, 0, 0, 0);
        };
        one(2, 0); one(1, 1); one(0, 2); one(1, 0); one(0, 1); one(0, 0);
        return c;
    }
};
struct ProductI8 {
    typedef pccnn_i32x16 Acc;
    static constexpr int TERMS = 1, UNIT = 16, UNITS = 8;
    static __device__ __forceinline__ Acc mma(const pccnn_u32x4 (&a)[1], const pccnn_u32x4 (&b)[1], Acc c)
    {
        return __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(pccnn_i32x4, a[0]), __builtin_bit_cast(pccnn_i32x4, b[0]),
                                                     c, 0, 0, 0);
    }
};

// A window whose base the compiler takes as the same in all lanes, which it cannot always see.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t product_window(const void *base)
{
    const uint64_t bits = (uint64_t)base;
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)bits), hi = __builtin_amdgcn_readfirstlane((uint32_t)(bits >> 32));
    return attn_window((const void *)((uint64_t)hi << 32 | lo));
}

// quotient and rest of a workgroup's number, in scalar registers (the division itself runs in vector ones).
__device__ __forceinline__ uint32_t product_split(uint32_t &block, uint32_t by)
{
    const uint32_t quotient = __builtin_amdgcn_readfirstlane(block / by), rest = block - quotient * by;
    block = quotient;
    return rest;
}

// f32 values from their terms (attn_split): the terms' sum is exact.
__device__ __forceinline__ float product_value(float t0, float t1, float t2) { return fabsf(t1) <= FLT_MAX ? t2 + t1 + t0 : t1; }
// Unit `unit` of an operand row of three planes; zeros from `units` on.
__device__ __forceinline__ void product_values(const ProductRows &s, int64_t row, int unit, int units, float (&v)[8])
{
    float t[3][8];
#pragma unroll
    for (int i = 0; i < 8; ++i) t[0][i] = t[1][i] = t[2][i] = 0.0f;
    if (unit < units) {
        const char *at = (const char *)s.p + row * s.stride + unit / 8 * s.step + unit % 8 * 16;
#pragma unroll
        for (int i = 0; i < 3; ++i) pccnn_load<8>((const uint16_t *)(at + i * s.plane), t[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = product_value(t[0][i], t[1][i], t[2][i]);
}
// The largest magnitude of a block's results; NaN if there is one.  An instruction for two of them (inference 400000 x 64 -> 176
// 245 us, unsettled 235, with a comparison for each 253).
template <int COUNT, typename ACC> __device__ __forceinline__ float product_most(const ACC &acc)
{
    float most = 0.0f;
#pragma unroll
    for (int e = 0; e < COUNT; e += 2)
        most = __builtin_elementwise_maximum(__builtin_elementwise_maximum(most, fabsf(acc[e])), fabsf(acc[e + 1]));
    return most;
}
__device__ __forceinline__ bool product_unsettled(float most) { return __any(!(most <= FLT_MAX)); }

// Brings tile after tile of ROWS operand rows, UNITS units of 16 bytes of each, into LDS: the inner dimension lies along the rows.
// TERMS tiles, one of each plane, one behind the other.
template <int ROWS, int THREADS, int UNITS, int TERMS> struct RowsFeeder {
    typedef AttnTile<1, ROWS, 8 * UNITS> Tile;
    static constexpr int ROUNDS = (ROWS * UNITS + THREADS - 1) / THREADS, COUNT = ROUNDS * TERMS;     // requests of a wavefront
    static constexpr int ELEMENTS = TERMS * Tile::PLANE;
    static_assert(THREADS / UNITS % 16 == 0 && ROWS * UNITS % PCCNN_WAVE == 0 && (ROUNDS == 1 || ROUNDS * THREADS == ROWS * UNITS),
                  "whole wavefronts, the same unit in every round");
    const char *base, *at;                   // the tile's first row, and of it what is asked for next (the same in all lanes)
    int64_t plane, step;
    uint32_t off[ROUNDS];                    // the lane's units from there, in bytes
    int unit;                                // which of a row's units the lane brings
    bool mine, second;                       // this wavefront brings any (tiles of few rows); UNITS 4: the second half is next
    __device__ __forceinline__ void start(const ProductRows &s, int64_t row)
    {
        at = (const char *)s.p + row * s.stride;
        plane = s.plane;
        step = s.step;
        second = false;
        const int r = (int)threadIdx.x / UNITS, stride = (int)s.stride, left = (int)min(s.rows - row, (int64_t)ROWS);
        unit = Tile::unit_at(r % ROWS, (int)threadIdx.x % UNITS);
        mine = ROWS * UNITS >= THREADS || __builtin_amdgcn_readfirstlane(threadIdx.x) < ROWS * UNITS;
        const uint32_t first = r * stride + 16 * unit;
#pragma unroll
        for (int j = 0; j < ROUNDS; ++j)
            off[j] = r + j * (THREADS / UNITS) < left ? first + j * (THREADS / UNITS * stride) : kAttnNowhere;
    }
    // The next units of every row; `units`: how many of them exist.  A tile comes in ALL requests of a wavefront, of which this
    // operand's are those from FIRST on; `part`: which half of them.
    template <int FIRST, int ALL> __device__ __forceinline__ void fetch(int part, int units, uint16_t *tile) const
    {
        if (!mine) return;
        const int wave_unit = __builtin_amdgcn_readfirstlane(threadIdx.x & ~(PCCNN_WAVE - 1));
#pragma unroll
        for (int t = 0; t < TERMS; ++t) {
            const __amdgpu_buffer_rsrc_t window = product_window(at + t * plane);
#pragma unroll
            for (int j = 0; j < ROUNDS; ++j)
                if ((FIRST + t * ROUNDS + j) * 2 / ALL == part)
                    attn_bring(window, unit < units ? off[j] : kAttnNowhere, tile + t * Tile::PLANE + 8 * (j * THREADS + wave_unit));
        }
    }
    __device__ __forceinline__ void next()
    {
        if constexpr (UNITS == 8) {
            at += step;
        } else {                             // the other half of 128 bytes, then on
            at += second ? step - 64 : 64;
            second = !second;
        }
    }
};

// What this wavefront asked for, but for the newest BUT requests, has landed and its reads of LDS are done; behind the barrier,
// those of the workgroup.
template <int BUT = 0> __device__ __forceinline__ void product_landed()
{
    static_assert(BUT < 64, "a count of six bits");
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((BUT & 15) | (BUT >> 4) << 14 | 0x0070);                // vmcnt(BUT) lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// The product of BM rows of the lane's side with BN rows of the registers' side, both with the inner dimension along the rows.
// WM x WN wavefronts, each with MT x NT blocks of 32 x 32.  PAIR: the registers' side is BN / 2 rows of one operand and as many
// of another (gate and up), and the first half of a wavefront's NT blocks is of the first, the second half of the second, of the
// same channels.  Two tiles are in LDS, one worked on while the next is brought; three of 64 rows, of which a launch has few, so that
// a tile is asked for two steps ahead (gradients 1000 x 512 -> 1408 bf16 81.6 -> 72.4 us, f32 161 -> 145; four are no better).
template <class E, int BM, int BN, int WM, int WN, bool PAIR> struct ProductNT {
    static constexpr int THREADS = WM * WN * PCCNN_WAVE, MT = BM / WM / 32, NT = BN / WN / 32;
    static constexpr int TERMS = E::TERMS, UNITS = E::UNITS, STEPS = UNITS / 2;       // products of sixteen bf16 to a tile
    static constexpr int PART = PAIR ? BN / 2 : BN;                   // rows of one operand of the registers' side
    typedef RowsFeeder<BM, THREADS, UNITS, TERMS> FeedM;
    typedef RowsFeeder<PART, THREADS, UNITS, TERMS> FeedN;
    static constexpr int STAGE = FeedM::ELEMENTS + (PAIR ? 2 : 1) * FeedN::ELEMENTS;  // uint16_t
    static constexpr int STAGES = BM == 64 ? 3 : 2;
    static_assert(STAGES == 2 || (BM * UNITS >= THREADS && PART * UNITS >= THREADS), "all wavefronts ask as often");
    static constexpr size_t lds_bytes(int units)                      // (no more tiles than there are steps)
    {
        return (size_t)std::min((units + UNITS - 1) / UNITS, STAGES) * STAGE * sizeof(uint16_t);
    }
    typename E::Acc acc[MT][NT];
    int lane, half, wm, wn;
    __device__ __forceinline__ ProductNT()
    {
        lane = threadIdx.x % PCCNN_WAVE;
        half = lane >> 5;
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / PCCNN_WAVE);
        wm = wave % WM;
        wn = wave / WM;
    }
    // Tile row of the lane's side of block m; first tile row of the registers' side of block n.
    __device__ __forceinline__ int row_of(int m) const { return wm * (32 * MT) + 32 * m + (lane & 31); }
    __device__ __forceinline__ int col_of(int n) const
    {
        if constexpr (PAIR) return n / (NT / 2) * PART + wn * (16 * NT) + 32 * (n % (NT / 2));
        return wn * (32 * NT) + 32 * n;
    }
    // One tile's products, and among their first half, in two parts, what `ask` asks memory for.  A compute unit takes a request
    // of a wavefront every sixteen cycles, so eight wavefronts that ask for a whole tile at once wait for each other; what is
    // asked for in the second half is late for the next tile.  65536 x 2816 x 512: at once 196 us, four parts over the whole 205,
    // two parts over the first half 197; 65536 x 512 x 512 40.1, 40.6 and 39.3, 65536 x 1408 x 512 83.7, 85.0 and 81.2.
    // BEGIN: the first tile, whose first products begin the sums (clearing the registers would cost two instructions a result,
    // a tenth of what a gelu takes).
    template <bool BEGIN, typename ASK> __device__ __forceinline__ void multiply(const uint16_t *tile, ASK ask)
    {
        const typename E::Acc zero = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
        typedef typename FeedM::Tile TileM;
        typedef typename FeedN::Tile TileN;
        uint16_t *const tm = const_cast<uint16_t *>(tile), *const tn = tm + FeedM::ELEMENTS;
        // operands are read a step of products ahead of their use: the compiler, left alone, reads them just before
        pccnn_u32x4 a[2][NT][TERMS], b[2][MT][TERMS];
        auto read = [&](int kk) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int t = 0; t < TERMS; ++t) {
                    const int col = col_of(n), which = col / PART;    // gate or up: one behind the other, each with its planes
                    a[kk & 1][n][t] = __builtin_bit_cast(
                        pccnn_u32x4, TileN{tn + (which * TERMS + t) * TileN::PLANE}.rows(col % PART + (lane & 31), 2 * kk + half).t[0]);
                }
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int t = 0; t < TERMS; ++t)
                    b[kk & 1][m][t] =
                        __builtin_bit_cast(pccnn_u32x4, TileM{tm + t * TileM::PLANE}.rows(row_of(m), 2 * kk + half).t[0]);
        };
        read(0);
#pragma unroll
        for (int kk = 0; kk < STEPS; ++kk) {
            if (kk + 1 < STEPS) read(kk + 1);
            __builtin_amdgcn_sched_barrier(0x6);                      // VALU and SALU may cross
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int m = 0; m < MT; ++m) acc[m][n] = E::mma(a[kk & 1][n], b[kk & 1][m], BEGIN && kk == 0 ? zero : acc[m][n]);
                if (n == 0 && kk < 2) {
                    __builtin_amdgcn_sched_barrier(0x6);
                    ask(kk);
                    __builtin_amdgcn_sched_barrier(0x6);
                }
            }
            __builtin_amdgcn_sched_barrier(0x6);
        }
    }
    // Rows from `row` of `x`, rows from `col` of `one` (and `two`); `units`: 16-byte units of every row, at least one.
    // `last(there)` is called among the products of the last tile, when nothing is asked for any more: `there` is a tile's room in LDS
    // that nobody uses, and what is asked for into it is there on return.  Returns that room.
    template <typename LAST>
    __device__ __forceinline__ uint16_t *run(const ProductRows &x, int64_t row, const ProductRows &one, const ProductRows &two,
                                             int64_t col, int units, uint16_t *lds, LAST last)
    {
        FeedM fm;
        FeedN f1, f2;
        fm.start(x, row);
        f1.start(one, col);
        if constexpr (PAIR) f2.start(two, col);
        int left = units;                                             // of the tile that is asked for next
        const int total = (units + UNITS - 1) / UNITS;
        constexpr int ALL = FeedM::COUNT + (PAIR ? 2 : 1) * FeedN::COUNT;
        auto fetch = [&](int part, uint16_t *to) {
            fm.template fetch<0, ALL>(part, left, to);
            f1.template fetch<FeedM::COUNT, ALL>(part, left, to + FeedM::ELEMENTS);
            if constexpr (PAIR)
                f2.template fetch<FeedM::COUNT + FeedN::COUNT, ALL>(part, left, to + FeedM::ELEMENTS + FeedN::ELEMENTS);
            if (part == 0) return;
            left -= UNITS;
            fm.next();
            f1.next();
            if constexpr (PAIR) f2.next();
        };
#pragma unroll
        for (int i = 0; i < STAGES - 1; ++i)
            if (i < total) {
                fetch(0, lds + i * STAGE);
                fetch(1, lds + i * STAGE);
            }
        // `here` holds what is worked on, `there` is where the next tile goes.  That the two do not overlap is what lets the reads go
        // on while the tile is on its way.
        auto walk = [&](auto begin, const uint16_t *__restrict__ here, uint16_t *__restrict__ there, bool more, bool end) {
            multiply<decltype(begin)::value>(here, [&](int part) {
                if (more)
                    fetch(part, there);
                else if (end && part == 0)
                    last(there);
            });
        };
        // the tile that is worked on next; `newer`: tiles behind it that have been asked for
        auto landed = [&](int newer) {
            if constexpr (STAGES > 2)
                if (newer > 0) return product_landed<ALL>();
            product_landed();
        };
        landed(min(total, STAGES - 1) - 1);
        int slot = 0, free = total == 1 ? 1 : STAGES - 1;
        walk(std::true_type(), lds, lds + free * STAGE, total >= STAGES, total == 1);
        for (int step = 1; step < total; ++step) {
            landed(min(total - step, STAGES - 1) - 1);
            free = slot;                                              // the tile of the step before
            slot = slot + 1 < STAGES ? slot + 1 : 0;
            walk(std::false_type(), lds + slot * STAGE, lds + free * STAGE, step + STAGES <= total, step + 1 == total);
        }
        product_landed();                                             // LDS is free for the results
        return lds + free * STAGE;
    }
    __device__ __forceinline__ void run(const ProductRows &x, int64_t row, const ProductRows &one, const ProductRows &two,
                                        int64_t col, int units, uint16_t *lds)
    {
        run(x, row, one, two, col, units, lds, [](uint16_t *) {});
    }
    // Behind `run`, with the same arguments: f32 results that are not finite, again.  (Rows and channels that do not exist take the
    // last one's values.)  32000 x 512 -> 1408: 0.61 to 0.66 ms, with one infinite weight no more, with a column of them 1.53.
    __device__ __forceinline__ void settle(const ProductRows &x, int64_t row, const ProductRows &one, const ProductRows &two, int64_t col,
                                           int units)
    {
        if constexpr (TERMS == 3) {
            float most = 0.0f;
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int n = 0; n < NT; ++n) most = __builtin_elementwise_maximum(most, product_most<16>(acc[m][n]));
            if (!product_unsettled(most)) return;
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    if (!product_unsettled(product_most<16>(acc[m][n]))) continue;
                    const ProductRows &w = PAIR && n >= NT / 2 ? two : one;
                    const int64_t x_row = min(row + row_of(m), x.rows - 1);
                    const int64_t w_row = min(col + col_of(n) % PART + (lane & 31), w.rows - 1);
                    pccnn_f32x16 again = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll 1
                    for (int unit = 0; unit < units; unit += 2) {     // a unit for each half of the wavefront
                        float a[8], b[8];
                        product_values(w, w_row, unit + half, units, a);
                        product_values(x, x_row, unit + half, units, b);
#pragma unroll
                        for (int i = 0; i < 8; ++i) again = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], again, 0, 0, 0);
                    }
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (!(fabsf(acc[m][n][e]) <= FLT_MAX)) acc[m][n][e] = again[e];
                }
        }
    }
};

// A tile of BM rows of COLS results in LDS, on its way between the lanes that computed it and whole lines of memory.  The 16-byte
// units of a row are exchanged among themselves by the row, since 32 lanes write the same columns of 32 rows.
template <typename T, int BM, int COLS, int THREADS> struct ProductStage {
    static constexpr int PER = 16 / sizeof(T), UNITS = COLS / PER;
    static constexpr size_t BYTES = (size_t)BM * COLS * sizeof(T);
    T *base;
    static __device__ __forceinline__ int place(int row, int unit) { return unit ^ (row & (UNITS < 8 ? UNITS - 1 : 7)); }
    __device__ __forceinline__ T *at(int row, int col) const
    {
        return base + row * COLS + PER * place(row, col / PER) + col % PER;
    }
    // Columns col .. col + 3 (col a multiple of four) of a row.
    __device__ __forceinline__ void put(int row, int col, const float (&v)[4]) const { pccnn_store<4>(at(row, col), v); }
    __device__ __forceinline__ void get(int row, int col, float (&v)[4]) const { pccnn_load<4>(at(row, col), v); }
    // Rows row0 .. of `from`, columns col0 .. , zeros past `rows` and `width`.  Rows that are whole 16-byte units: lands by the next
    // wait for vector memory.
    __device__ __forceinline__ void bring(const T *from, int64_t stride, int64_t row0, int64_t rows, int64_t col0, int64_t width) const
    {
        constexpr int COUNT = BM * UNITS / THREADS;
        static_assert(COUNT * THREADS == BM * UNITS && THREADS % (8 * UNITS) == 0, "the same unit in every round");
        const int r0 = (int)threadIdx.x / UNITS, unit = place(r0, (int)threadIdx.x % UNITS);
        const int64_t col = col0 + unit * PER;
        const __amdgpu_buffer_rsrc_t window = product_window(from + row0 * stride + col0);
        const int wave_unit = __builtin_amdgcn_readfirstlane(threadIdx.x & ~(PCCNN_WAVE - 1));
#pragma unroll
        for (int j = 0; j < COUNT; ++j) {
            const int r = r0 + j * (THREADS / UNITS);
            attn_bring(window, row0 + r < rows && col < width ? (uint32_t)((r * stride + unit * PER) * sizeof(T)) : kAttnNowhere,
                       base + PER * (j * THREADS + wave_unit));
        }
    }
    // The same of rows that are not; needs a barrier behind it.
    __device__ __forceinline__ void copy(const T *from, int64_t stride, int64_t row0, int64_t rows, int64_t col0, int64_t width) const
    {
        for (int i = threadIdx.x; i < BM * UNITS; i += THREADS) {
            const int r = i / UNITS, unit = i % UNITS;
#pragma unroll
            for (int e = 0; e < PER; ++e) {
                const int64_t col = col0 + unit * PER + e;
                base[r * COLS + PER * place(r, unit) + e] = row0 + r < rows && col < width ? from[(row0 + r) * stride + col] : (T)0;
            }
        }
    }
    // Writes the tile to `to`'s rows, columns below `width`, as whole units where every row allows it.  A thread has the same unit of
    // every THREADS / UNITS-th row.
    template <typename ROW> __device__ __forceinline__ void out(const ROW &to, int64_t row0, int64_t rows, int64_t col0, int64_t width) const
    {
        constexpr int COUNT = BM * UNITS / THREADS, EVERY = THREADS / UNITS;
        static_assert(COUNT * THREADS == BM * UNITS && EVERY % 8 == 0, "the same unit in every round");
        const int r0 = (int)threadIdx.x / UNITS, unit = (int)threadIdx.x % UNITS;
        const int64_t col = col0 + unit * PER;
        const int left = (int)min(rows - row0, (int64_t)BM);
        if (col >= width) return;
        const T *from = base + r0 * COLS + PER * place(r0, unit);
        T *at = to.at(row0 + r0, col);
        const int64_t step = EVERY * to.row_step();
        if (to.lines()) {                    // whole lines that no kernel of the call reads again: past the caches (see below)
#pragma unroll
            for (int j = 0; j < COUNT; ++j, at += step)
                if (r0 + j * EVERY < left)
                    __builtin_nontemporal_store(*(const pccnn_u32x4 *)(from + j * EVERY * COLS), (pccnn_u32x4 *)at);
        } else if (to.whole() && width % PER == 0) {
#pragma unroll
            for (int j = 0; j < COUNT; ++j, at += step)
                if (r0 + j * EVERY < left) *(pccnn_u32x4 *)at = *(const pccnn_u32x4 *)(from + j * EVERY * COLS);
        } else {
            for (int j = 0; j < COUNT; ++j, at += step)
                if (r0 + j * EVERY < left)
#pragma unroll
                    for (int e = 0; e < PER; ++e)
                        if (col + e < width) at[e] = from[j * EVERY * COLS + e];
        }
    }
};
// Where a unit of a result lies, and whether it goes past the caches.  Results whose rows are whole lines do (800000 x 64 -> 256
// 159 -> 144 us, 34123 x 512 -> 1408 in 8 bits 86 -> 79); partial lines do not (34123 x 1000 f32 49 -> 54), nor does what the next
// kernels read (training 8192 x 512 -> 1408 174 -> 182, 400000 x 64 -> 176 341 -> 368; 65536 x 512 -> 1408 832 -> 823; dx in parts,
// 300 x 512 -> 1408 f32 70.0 -> 70.8, bf16 41.9 -> 42.1).
// Rows of `stride` elements; or pieces of 64 columns of all rows, one behind the other, so that what a tile of rows takes of one
// piece lies together (65536 x 2816 x 512: 167 us, with rows in one piece 196; 65536 x 512 under 2816 columns, the inner
// dimension over the rows, 191 and 219).
template <typename T> struct DenseRow {
    T *p;
    int64_t stride;
    bool read_next = false;                  // by the call's next kernel
    __device__ __forceinline__ bool whole() const { return stride * (int)sizeof(T) % 16 == 0; }
    __device__ __forceinline__ bool lines() const { return !read_next && stride * (int)sizeof(T) % 128 == 0; }
    __device__ __forceinline__ int64_t row_step() const { return stride; }
    __device__ __forceinline__ T *at(int64_t row, int64_t col) const { return p + row * stride + col; }
};
template <typename T> struct PieceRow {
    T *p;
    int64_t rows, from;                      // `from`: the column of all pieces that column 0 is
    __device__ __forceinline__ bool whole() const { return true; }
    __device__ __forceinline__ bool lines() const { return false; }  // (the next kernels read it)
    __device__ __forceinline__ int64_t row_step() const { return 64; }
    __device__ __forceinline__ T *at(int64_t row, int64_t col) const
    {
        return p + ((from + col) / 64 * rows + row) * 64 + (from + col) % 64;
    }
};

// What belongs to the tile's output channels (scales, a bias), in LDS before the products begin: COUNT arrays of COLS values, those
// of channels that do not exist zero.  There by the first barrier.
template <int COUNT, int COLS, int THREADS> struct ProductChannels {
    static constexpr size_t BYTES = COUNT * COLS * sizeof(float);
    float *base;
    __device__ __forceinline__ void start(int which, const float *from, int64_t col0, int64_t cols) const
    {
        for (int i = threadIdx.x; i < COLS; i += THREADS)
            base[which * COLS + i] = from != nullptr && col0 + i < cols ? from[col0 + i] : 0.0f;
    }
    __device__ __forceinline__ void get(int which, int col, float (&v)[4]) const { pccnn_load<4>(base + which * COLS + col, v); }
};

// ---------------------------------------------------------------------------------------------- few rows
//
// Few rows (32 or 64 at most): no tile is shared by enough of them to be worth LDS.  A workgroup has sixteen output channels (of one
// or two operands); its wavefronts deal the inner dimension among themselves in steps of 64 bytes, take weights and rows from memory
// straight into operands of 16 x 16 products, and add their sums in LDS in a fixed order.
template <typename T> struct FewStep;                                // elements of a lane's operand, of a step of four lanes
template <> struct FewStep<uint16_t> { static constexpr int UNIT = 8, TERMS = 1; typedef pccnn_f32x4 Acc; typedef float Sum; };
template <> struct FewStep<float> { static constexpr int UNIT = 8, TERMS = 3; typedef pccnn_f32x4 Acc; typedef float Sum; };
template <> struct FewStep<int8_t> { static constexpr int UNIT = 16, TERMS = 1; typedef pccnn_i32x4 Acc; typedef int Sum; };

template <int TERMS> struct FewFrag { pccnn_u32x4 t[TERMS]; };

template <typename T> __device__ __forceinline__ FewFrag<FewStep<T>::TERMS> few_load(const T *row, int64_t col, int64_t width, int wide)
{
    FewFrag<FewStep<T>::TERMS> f;
    if constexpr (std::is_same<T, int8_t>::value) {
        f.t[0] = (pccnn_u32x4){0u, 0u, 0u, 0u};
        if (col < width) {
            if (wide == 2) {
                f.t[0] = *(const pccnn_u32x4 *)(row + col);
            } else if (wide == 1) {          // (rows of whole four bytes)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (col + 4 * i < width) f.t[0][i] = *(const uint32_t *)(row + col + 4 * i);
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (col + i < width) f.t[0][i / 4] |= (uint32_t)(uint8_t)row[col + i] << (8 * (i % 4));
            }
        }
    } else {
        AttnChunk<T> c;
        attn_load(c, row, (int)col, (int)width, wide);
        const auto g = attn_frag(c);
#pragma unroll
        for (int t = 0; t < FewStep<T>::TERMS; ++t) f.t[t] = __builtin_bit_cast(pccnn_u32x4, g.t[t]);
    }
    return f;
}
template <typename T>
__device__ __forceinline__ void few_mma(typename FewStep<T>::Acc &c, const FewFrag<FewStep<T>::TERMS> &a,
                                        const FewFrag<FewStep<T>::TERMS> &b)
{
    if constexpr (std::is_same<T, int8_t>::value) {
        c = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(pccnn_i32x4, a.t[0]), __builtin_bit_cast(pccnn_i32x4, b.t[0]),
                                                  c, 0, 0, 0);
    } else {
        auto one = [&](int i, int j) {
            c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pccnn_bf16x8, a.t[i]),
                                                        __builtin_bit_cast(pccnn_bf16x8, b.t[j]), c, 0, 0, 0);
        };
        if constexpr (FewStep<T>::TERMS == 3) {
            one(2, 0); one(1, 1); one(0, 2); one(1, 0); one(0, 1);
        }
        one(0, 0);
    }
}

struct FewRows {
    const void *p;
    int64_t stride;                          // elements
    int wide;
};
// Sums of sixteen output channels from `col` of OUTS operands with RT x 16 rows, in the first wavefront's registers: lane & 15 is
// the row, 4 (lane / 16) + i the channel.  False in the other wavefronts.
template <typename T, int OUTS, int RT, int WAVES> struct FewProduct {
    typedef FewStep<T> S;
    typename S::Acc acc[RT][OUTS];
    __device__ __forceinline__ bool run(const FewRows &x, int64_t rows, const FewRows (&w)[OUTS], int64_t col, int64_t cols,
                                        int64_t inner, pccnn_u32x4 (*lds)[RT * OUTS][PCCNN_WAVE])
    {
        const int lane = threadIdx.x % PCCNN_WAVE, wave = threadIdx.x / PCCNN_WAVE;
        const int line = lane & 15, quarter = lane >> 4;
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int o = 0; o < OUTS; ++o) acc[r][o] = (typename S::Acc){0, 0, 0, 0};
        const T *xr[RT], *wr[OUTS];
        // rows and channels that do not exist take the last one's values, and nobody reads their sums
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            const int64_t row = 16 * r + line;
            xr[r] = (const T *)x.p + (row < rows ? row : rows - 1) * x.stride;
        }
#pragma unroll
        for (int o = 0; o < OUTS; ++o) wr[o] = (const T *)w[o].p + (col + line < cols ? col + line : cols - 1) * w[o].stride;
        for (int64_t k = (int64_t)wave * 4 * S::UNIT; k < inner; k += WAVES * 4 * S::UNIT) {
            const int64_t at = k + quarter * S::UNIT;
            FewFrag<S::TERMS> a[OUTS], b[RT];
#pragma unroll
            for (int o = 0; o < OUTS; ++o) a[o] = few_load<T>(wr[o], at, inner, w[o].wide);
#pragma unroll
            for (int r = 0; r < RT; ++r) b[r] = few_load<T>(xr[r], at, inner, x.wide);
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int o = 0; o < OUTS; ++o) few_mma<T>(acc[r][o], a[o], b[r]);
        }
        if (wave > 0)
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int o = 0; o < OUTS; ++o) lds[wave - 1][r * OUTS + o][lane] = __builtin_bit_cast(pccnn_u32x4, acc[r][o]);
        __syncthreads();
        if (wave > 0) return false;
        for (int v = 0; v < WAVES - 1; ++v)
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int o = 0; o < OUTS; ++o)
                    acc[r][o] += __builtin_bit_cast(typename S::Acc, lds[v][r * OUTS + o][lane]);
        if constexpr (std::is_same<T, float>::value) settle(x, rows, w, col, cols, inner, lds[0]);
        return true;
    }
    // As ProductNT::settle has it; one block after the other, in `lds`, so that the sums' registers are all that it adds to the way of
    // the others.
    __device__ __forceinline__ void settle(const FewRows &x, int64_t rows, const FewRows (&w)[OUTS], int64_t col, int64_t cols,
                                           int64_t inner, pccnn_u32x4 (*lds)[PCCNN_WAVE])
    {
        float most = 0.0f;
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int o = 0; o < OUTS; ++o) most = __builtin_elementwise_maximum(most, product_most<4>(acc[r][o]));
        if (!product_unsettled(most)) return;
        const int lane = threadIdx.x % PCCNN_WAVE, line = lane & 15, quarter = lane >> 4;
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int o = 0; o < OUTS; ++o) lds[r * OUTS + o][lane] = __builtin_bit_cast(pccnn_u32x4, acc[r][o]);
#pragma unroll 1
        for (int block = 0; block < RT * OUTS; ++block) {
            pccnn_f32x4 c = __builtin_bit_cast(pccnn_f32x4, lds[block][lane]), again = {0, 0, 0, 0};
            const FewRows &one = w[block % OUTS];
            const float *xr = (const float *)x.p + min((int64_t)(16 * (block / OUTS) + line), rows - 1) * x.stride;
            const float *wr = (const float *)one.p + min(col + line, cols - 1) * one.stride;
#pragma unroll 1
            for (int k = 0; k < (int)inner; k += 4 * S::UNIT) {
                AttnChunk<float> a, b;
                attn_load(a, wr, k + quarter * S::UNIT, (int)inner, one.wide);
                attn_load(b, xr, k + quarter * S::UNIT, (int)inner, x.wide);
#pragma unroll
                for (int i = 0; i < S::UNIT; ++i) again = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[i], b.v[i], again, 0, 0, 0);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (!(fabsf(c[e]) <= FLT_MAX)) c[e] = again[e];
            lds[block][lane] = __builtin_bit_cast(pccnn_u32x4, c);
        }
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int o = 0; o < OUTS; ++o) acc[r][o] = __builtin_bit_cast(typename S::Acc, lds[r * OUTS + o][lane]);
    }
};

// ---------------------------------------------------------------------------------------------- operands laid out
//
// Rows of `width` elements, `stride` apart, as rows of whole 16-byte units with zeros behind the last element; f32 as three planes
// of bf16 terms, `plane` elements apart.  Up to three tensors in one launch (blockIdx.y), a unit per thread.
struct StageSource {
    const void *p;
    int64_t stride, rows;
    int wide;
    void *to;
};
struct StageArgs {
    StageSource s[3];
    int64_t width;
    int units;
};
template <typename T> __device__ __forceinline__ void product_stage(const StageArgs &a, uint32_t which, uint32_t block, uint32_t blocks)
{
    constexpr int UNIT = FewStep<T>::UNIT, TERMS = FewStep<T>::TERMS;
    const StageSource s = which == 0 ? a.s[0] : which == 1 ? a.s[1] : a.s[2];
    const int64_t count = s.rows * a.units;
    for (int64_t i = (int64_t)block * 256 + threadIdx.x; i < count; i += (int64_t)blocks * 256) {
        const int64_t row = i / a.units;
        const FewFrag<TERMS> f = few_load<T>((const T *)s.p + row * s.stride, (i - row * a.units) * UNIT, a.width, s.wide);
#pragma unroll
        for (int t = 0; t < TERMS; ++t) ((pccnn_u32x4 *)s.to)[t * count + i] = f.t[t];
    }
}
template <typename T> static __global__ __launch_bounds__(256) void product_stage_kernel(StageArgs a)
{
    product_stage<T>(a, blockIdx.y, blockIdx.x, gridDim.x);
}
static inline unsigned product_stage_blocks(int64_t units) { return (unsigned)std::min<int64_t>(pccnn_ceil_div(units, 256), 8192); }

// ---------------------------------------------------------------------------------------------- launches
//
// Tiles of 256 x 256 (one workgroup of eight wavefronts to a CU) rather than 128 x 128: for sums of 512 terms and more where the
// last round of workgroups leaves no more than 15 % of all rounds idle.  Gated maps in us, 256 x 256 against 128 x 128:
// 32000 x 512 -> 1408 bf16 102 : 108, in 8 bits 79 : 82; 8000 x 1024 -> 2800 (0.92 of the rounds filled) 99 : 111, 8 bits 68 : 72;
// not for 8000 x 512 -> 1408 (0.69 of them) 34 : 30, 8 bits 27 : 22, nor for 256 terms, 32000 x 256 -> 704 36 : 34.
static inline bool product_large(int64_t rows, int64_t cols, int64_t depth)
{
    const int64_t tiles = pccnn_ceil_div(rows, 256) * pccnn_ceil_div(cols, 256);
    return depth >= 512 && cols >= 256 && tiles * 20 >= pccnn_ceil_div(tiles, 256) * 256 * 17;
}
// Tiles of 64 x 64 rather than 128 x 128 where those leave compute units without work.  In us, 64 x 64 against 128 x 128: 88 tiles
// of 128 (1000 x 256 -> 704) bf16 5.1 : 5.6, 8 bits 5.0 : 5.7, f32 18.2 : 20.3; 176 of them (1000 x 512 -> 1408) 9.1 : 8.1,
// 6.8 : 6.9, 51 : 36; 192 (4000 x 128 -> 344) 5.2 : 5.2, 5.1 : 5.5, 15.5 : 15.1.
static inline bool product_small(int64_t rows, int64_t cols) { return pccnn_ceil_div(rows, 128) * pccnn_ceil_div(cols, 128) < 160; }
template <typename KERNEL, typename ARGS>
static int product_launch(const char *name, KERNEL kernel, size_t lds, int threads, ARGS &a, int64_t tiles_m, int64_t tiles_n,
                          hipStream_t s)
{
    // (a launch has less than 2^32 threads)
    PCCNN_REQUIRE(tiles_m * tiles_n <= (int64_t)UINT32_MAX / threads - 1024, PCCNN_ERR_UNSUPPORTED, "%s: %lld workgroups", name,
                  (long long)(tiles_m * tiles_n));
    a.grid = product_grid(tiles_m, tiles_n);
    if (lds > 65536)
        PCCNN_HIP_CHECK(hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    kernel<<<product_workgroups(a.grid), threads, lds, s>>>(a);
    PCCNN_LAUNCH_CHECK();
    return PCCNN_OK;
}
#endif
