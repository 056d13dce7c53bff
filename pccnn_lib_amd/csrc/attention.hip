// Softmax attention of a cloud's queries to the keys of the same cloud at another level, forward and backward.
//
//   S = scale q . k   (minus infinity where the key is switched off)   P = softmax over the cloud's keys   O = P v
//   L = log sum exp S, kept for the backward pass:   P = exp(S - L)   D = dO . O   dS = P (dO . v - D)
//   dv = P^T dO   dq = scale dS k   dk = scale dS^T q
//
// Clouds lie one behind the other (starts[c] .. starts[c + 1]); no tensor is padded.  Query heads that share a key head
// are rows of one problem (row = query * group + head in group), so keys and values are read once for the group and the
// sum of the shared head's gradient over its query heads is part of the product.  Scores are never written: a wavefront
// owns 32 rows (forward, dq) or 32 keys (dk, dv) and walks the other side in tiles of 64, with the running maximum and
// sum of the softmax in f32.  S is formed transposed (its column, a row of the problem, in the lane), which makes the
// softmax statistics two values per lane and lets P serve as an operand of the next product without leaving its lane
// (attention_tiles.h).  dq and dk / dv are two kernels that each recompute S: 7 products instead of 5, no atomics, the
// same bits from run to run.
//
// bf16: P and dS are rounded to bf16 as operands (but P of few rows, see attention_fwd_kernel), D is formed from the rounded
// output (but among few keys, see attention_dq_kernel), results are rounded once; all sums and the softmax are f32.
// f32: three bf16 terms per value, six products (attention_tiles.h).
//
// Tiles go from memory to LDS without passing registers, the next while one is worked on.  What bounds the large cases is
// the card's power: matrix pipe 40 - 59 % and vector ALU 45 - 78 % busy at 1.65 - 2.1 GHz of 2.4, LDS 20 - 35 % without a
// conflict.  Wave priorities and exponentials interleaved with the next products by hand changed nothing.  64 rows per
// wavefront, which halve the reads of LDS, are faster for even clouds of 64 features (8 x 256 rows over 100000 keys 605 -> 568
// us) and slower for uneven ones (8 x 8192 rows 216 -> 240) and at 128 features (6.8 -> 7.4 ms, one wavefront to a SIMD).
// Measured: forward 34123 x 100000, 4 heads of 128, 6.5 - 6.9 ms = 1013 - 1075 TFLOP/s; training 8 x 8192 rows over 2047 keys,
// uneven, 8 heads of 64: forward 169 - 202, dq with the rows' statistics 212 - 250, dk / dv 325 - 383 us; one row per cloud over
// 16 x 4096 keys 25 us = 5.4 TB/s and 4 for the join, over 10^6 keys 92 us = 5.6 TB/s and 10.
#include "attention_tiles.h"

#include <algorithm>
#include <float.h>
#include <math.h>

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / PCCNN_WAVE;
constexpr int kOwn = 32 * kWaves;            // rows (forward, dq) or keys (dk, dv) of a workgroup
constexpr int kMaxWidth = 128;
constexpr int64_t kMostTokens = 1ll << 32;   // queries x heads, keys x key heads
// Own tiles per cloud from which on f32 is turned into planes of terms first.  Measured with and without, 4 clouds of 4 heads
// over 2048 keys, forward in us: 64 features, 2 tiles 36 and 34, 6 tiles 58 and 56, 7 tiles 66 and 70, 24 tiles 159 and 178; 128
// features, 2 tiles 53 and 47, 6 tiles 106 and 116, 24 tiles 295 and 371; 32 features gain later, 7 tiles 47 and 44, 12 tiles 60
// and 59, 24 tiles 103 and 106.  dq, dk and dv have their crossing at 4 to 8 tiles of 64 to 128 features, 8 to 12 of 32.
constexpr int kPlanesFrom = 7;
constexpr float kLog2e = 1.44269504088896341f;

// Rows of the other side that are in LDS at a time, twice (one tile is brought in while the other is worked on).  Three
// terms of wide heads take half as many (64 or 128 features: 48 and 96 KiB of a CU's 160; 96 features do not divide evenly).
template <typename T, int DP> constexpr int attn_tile_rows()
{
    return AttnTerms<T>::value == 3 && (DP == 64 || DP == 128) ? 32 : 64;
}

// The side that is walked: rows `n` elements apart, heads `h`.  Either as the caller has it (`wide`: attn_load), or - bf16
// features whose rows are whole 16-byte units - as planes that go to LDS without passing through registers.
struct AttnStream {
    const void *p;
    int64_t n, h, plane;
    int wide, units;
};

struct AttnArgs {
    const void *q, *k, *v, *g, *o;           // a workgroup's own side: queries, keys, values, gradient of the output, O
    int64_t q_n, q_h, k_n, k_h, v_n, v_h, g_n, g_h;
    int wide_q, wide_k, wide_v, wide_g, wide_o;
    AttnStream one, two;                     // the walked side: keys and values, or queries and output gradients
    const int32_t *q_starts, *k_starts;
    const uint8_t *mask;
    int64_t m, n;
    int clouds, heads, key_heads, group, width;
    float scale;
    int tiles, splits, per_split;            // own tiles per cloud and head; parts of the other side and tiles in each
    int longest_first;                       // clouds in the order of what a workgroup has to walk
    int run;                                 // consecutive workgroups that go to one XCD, so that its L2 serves them
    int64_t blocks;                          // workgroups with work
    void *out;                               // forward: O; backward: dq
    float *lse;                              // [m, heads]
    float *shift, *delta;                    // [key_heads][m * group]: a row's L in units of log 2 (+inf: no keys), and D
    void *d_k, *d_v;
    float *part, *part_v;                    // [split][rows or keys][heads][width] f32, when splits > 1
    float2 *part_ml;                         // [split][m][heads] (maximum in units of log 2, sum)
};

// The part of the problem a workgroup works on: logical block = ((cloud * key_heads + head) * splits + split) * tiles + tile.
struct AttnBlock {
    int64_t q0, k0;                          // first query and key of the cloud
    int rows, keys;                          // rows = queries * group
    int head, split, tile;
    // The cloud with the r-th longest other side (`starts`), for up to 64 clouds: workgroups start in the order of their
    // numbers, and the long ones shall not be the last.
    static __device__ __forceinline__ int longest(const int32_t *starts, int clouds, int r)
    {
        const int lane = threadIdx.x % PCCNN_WAVE;
        const int mine = lane < clouds ? starts[lane + 1] - starts[lane] : -1;
        int before = 0;
        for (int j = 0; j < clouds; ++j) {
            const int other = __builtin_amdgcn_readlane(mine, j);
            before += other > mine || (other == mine && j < lane);
        }
        return __builtin_ctzll(__ballot(lane < clouds && before == r) | 1ull << 63);
    }
    __device__ __forceinline__ AttnBlock(const AttnArgs &a, int64_t block, const int32_t *walked)
    {
        tile = (int)(block % a.tiles);
        block /= a.tiles;
        split = (int)(block % a.splits);
        block /= a.splits;
        head = (int)(block % a.key_heads);
        int cloud = (int)(block / a.key_heads);
        if (a.longest_first) cloud = min(longest(walked, a.clouds, cloud), a.clouds - 1);
        // starts outside the tensors are a caller's mistake, but never an access outside them
        const int64_t q1 = min(max((int64_t)a.q_starts[cloud + 1], (int64_t)0), a.m);
        const int64_t k1 = min(max((int64_t)a.k_starts[cloud + 1], (int64_t)0), a.n);
        q0 = min(max((int64_t)a.q_starts[cloud], (int64_t)0), q1);
        k0 = min(max((int64_t)a.k_starts[cloud], (int64_t)0), k1);
        rows = (int)min((q1 - q0) * a.group, (int64_t)INT32_MAX - 2 * kOwn);
        keys = (int)(k1 - k0);
    }
    __device__ __forceinline__ int64_t query(const AttnArgs &a, int row) const { return q0 + row / a.group; }
    __device__ __forceinline__ int head_of(const AttnArgs &a, int row) const { return head * a.group + row % a.group; }
    // Where a row's shift and delta are.
    __device__ __forceinline__ int64_t stat(const AttnArgs &a, int row) const
    {
        return head * (a.m * a.group) + q0 * a.group + row;
    }
};

// One bit per row of a tile: the first `count` of `rows`.
__device__ __forceinline__ uint64_t first_bits(int count, int rows)
{
    return count <= 0 ? 0 : count >= rows ? (rows == 64 ? ~0ull : (1ull << rows) - 1) : (1ull << count) - 1;
}

// Which of the `rows` keys from `key` on take part: within the cloud and not switched off.  `flag` holds the lane's mask
// byte, loaded ahead of its use.
__device__ __forceinline__ uint8_t key_flag(const AttnArgs &a, const AttnBlock &b, int key, int lane)
{
    if (a.mask == nullptr) return 1;
    return key + lane < b.keys ? a.mask[b.k0 + key + lane] : 0;
}
__device__ __forceinline__ uint64_t live_keys(const AttnArgs &a, const AttnBlock &b, int key, uint8_t flag, int rows)
{
    const uint64_t all = first_bits(b.keys - key, rows);
    return a.mask == nullptr ? all : all & __ballot(flag != 0);
}

// Brings tile after tile of a stream into LDS.  GROUPED: a stream row is a row of the problem (query * group + head in
// group), else a key.  REPEAT: what lies past the last row is that row again instead of zeros (for queries: a zero times an
// infinite key would be NaN, where the row's own score is as good as any other for a probability that is zero anyway).
template <typename T, int DP, bool DIRECT, bool GROUPED, bool REPEAT = false> struct Feeder {
    static constexpr int TERMS = AttnTerms<T>::value;
    static constexpr int ROWS = attn_tile_rows<T, DP>();
    typedef AttnTile<TERMS, ROWS, DP> Tile;
    static constexpr int COUNT = ROWS * Tile::UNITS / kThreads;
    static_assert(COUNT >= 1 && COUNT * kThreads == ROWS * Tile::UNITS, "every thread carries whole units");
    const char *base;                        // DIRECT: the tile's first row (the same in all lanes)
    uint32_t off[DIRECT ? COUNT : 1];        // and from there the lane's units, in bytes
    int64_t step;
    AttnChunk<T> held[DIRECT ? 1 : COUNT];

    static __device__ __forceinline__ int row_of(int j) { return (threadIdx.x + j * kThreads) / Tile::UNITS; }
    static __device__ __forceinline__ int unit_of(int j) { return (threadIdx.x + j * kThreads) % Tile::UNITS; }
    static __device__ __forceinline__ int64_t offset(const AttnStream &s, int group, int row)
    {
        if constexpr (GROUPED) {
            const int query = group == 1 ? row : row / group;
            return query * s.n + (row - query * group) * s.h;
        } else {
            return row * s.n;
        }
    }
    // Tiles start at multiples of ROWS: where the group divides them, every tile has the same offsets within it.
    static __device__ __forceinline__ bool regular(int group) { return !GROUPED || ROWS % group == 0; }
    // `at`: the cloud's and head's first element.  Units past the heads' width lie nowhere, which reads zeros.
    __device__ __forceinline__ void start(const AttnStream &s, int64_t at, int group, int row)
    {
        if constexpr (DIRECT) {
            base = (const char *)s.p + 2 * (at + offset(s, group, row));
            step = 2 * (!GROUPED || group == 1 ? ROWS * s.n : ROWS / group * s.n);
#pragma unroll
            for (int j = 0; j < COUNT; ++j) {
                const int r = row_of(j), unit = Tile::unit_at(r, unit_of(j));
                off[j] = unit < s.units ? 2 * (uint32_t)(offset(s, group, r) + 8 * unit) : kAttnNowhere;
            }
        }
    }
    // Starts bringing the tile of rows `row` .. into `tile` (DIRECT), or into registers.  Rows without a bit in `live`
    // become zeros; `limit`: rows that exist; `masked`: other rows than the last ones may lack their bits.
    __device__ __forceinline__ void fetch(const AttnStream &s, int64_t at, int group, int row, int limit, uint64_t live,
                                          bool masked, int width, const Tile &tile)
    {
        if constexpr (DIRECT) {
            const bool past = REPEAT && limit - row < ROWS;
            if (!regular(group) || past) {               // the tile's first row may lie inside a group
                base = (const char *)s.p + 2 * (at + row / group * s.n);
#pragma unroll
                for (int j = 0; j < COUNT; ++j) {
                    const int unit = Tile::unit_at(row_of(j), unit_of(j)), r = REPEAT ? min(row_of(j), limit - row - 1) : row_of(j);
                    const int query = (row + r) / group, head = row + r - query * group;
                    if (unit < s.units) off[j] = 2 * (uint32_t)((query - row / group) * s.n + head * s.h + 8 * unit);
                }
            }
            uint32_t at_unit[COUNT];
            if (masked) {
#pragma unroll
                for (int j = 0; j < COUNT; ++j) at_unit[j] = (live >> row_of(j)) & 1 ? off[j] : kAttnNowhere;
            } else {
#pragma unroll
                for (int j = 0; j < COUNT; ++j) at_unit[j] = REPEAT || row_of(j) < limit - row ? off[j] : kAttnNowhere;
            }
            const int wave_unit = __builtin_amdgcn_readfirstlane(threadIdx.x & ~(PCCNN_WAVE - 1));
#pragma unroll
            for (int t = 0; t < TERMS; ++t) {
                const __amdgpu_buffer_rsrc_t window = attn_window(base + 2 * t * s.plane);
#pragma unroll
                for (int j = 0; j < COUNT; ++j)
                    attn_bring(window, at_unit[j], tile.base + t * Tile::PLANE + 8 * (j * kThreads + wave_unit));
            }
            base += step;
        } else {
#pragma unroll
            for (int j = 0; j < COUNT; ++j) {
                attn_clear(held[j]);
                const int r = REPEAT ? min(row + row_of(j), limit - 1) : row + row_of(j);
                if (r < limit) attn_load(held[j], (const T *)s.p + at + offset(s, group, r), 8 * unit_of(j), width, s.wide);
            }
        }
    }
    // Not DIRECT: what was fetched goes to LDS.
    __device__ __forceinline__ void put(const Tile &tile, uint64_t live) const
    {
        if constexpr (!DIRECT) {
#pragma unroll
            for (int j = 0; j < COUNT; ++j) {
                AttnChunk<T> chunk = held[j];
                if (!REPEAT && !((live >> row_of(j)) & 1)) attn_clear(chunk);
                tile.put(row_of(j), unit_of(j), attn_frag(chunk));
            }
        }
    }
};

// Sets scores of keys that do not take part to minus infinity (registers of C for the 32 keys from bit 0 of `live`).
__device__ __forceinline__ void hide(pccnn_f32x16 &s, uint32_t live, int half)
{
    const uint32_t mine = live >> (4 * half);
#pragma unroll
    for (int i = 0; i < 16; ++i)
        s[i] = (mine >> (8 * (i / 4) + i % 4)) & 1 ? s[i] : -INFINITY;
}

__device__ __forceinline__ void clear(pccnn_f32x16 &c)
{
#pragma unroll
    for (int i = 0; i < 16; ++i) c[i] = 0.0f;
}

// Registers 8 g .. 8 g + 7 of a tile of P or dS as an operand.
template <int TERMS> __device__ __forceinline__ AttnFrag<TERMS> half_of(const pccnn_f32x16 &s, int g)
{
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = s[8 * g + i];
    return attn_split<TERMS>(x);
}

// A lane's operand of its own side: DP features of one row in steps of sixteen, zeros where there is no row.
template <typename T, int DP>
__device__ __forceinline__ void own_side(AttnFrag<AttnTerms<T>::value> (&f)[DP / 16], const void *p, int64_t at, bool live,
                                         int half, int width, int wide)
{
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) {
        AttnChunk<T> c;
        attn_clear(c);
        if (live) attn_load(c, (const T *)p + at, 16 * kk + 8 * half, width, wide);
        f[kk] = attn_frag(c);
    }
}

// Writes a lane's column of a transposed result (features 32 dt + 8 (i / 4) + 4 half + i % 4 in register i) to a dense row.
template <typename T, int DP>
__device__ __forceinline__ void write_column(T *row, const pccnn_f32x16 (&acc)[DP / 32], float factor, int half, int width)
{
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int col = 32 * dt + 8 * q + 4 * half;
            float x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = acc[dt][4 * q + i] * factor;
            if (width % 4 == 0) {
                if (col < width) pccnn_store<4>(row + col, x);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float one[1] = {x[i]};
                    if (col + i < width) pccnn_store<1>(row + col + i, one);
                }
            }
        }
}

// f32 features as planes of their bf16 terms, [plane][token][head][DP], zeros past the width: what a walked side that
// several workgroups walk is turned into once, so that its tiles go to LDS as they are (9600 x 4 x 32 values of both
// tensors: 6 us).  Two tensors (blockIdx.y), one unit of eight features per thread.
template <int DP>
__global__ __launch_bounds__(kThreads) void attention_planes_kernel(AttnStream one, AttnStream two, int64_t tokens,
                                                                   int heads, int width, uint16_t *__restrict__ planes_one,
                                                                   uint16_t *__restrict__ planes_two)
{
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x, row = i / (DP / 8);
    if (row >= tokens * heads) return;
    const AttnStream &s = blockIdx.y == 0 ? one : two;
    uint16_t *to = (blockIdx.y == 0 ? planes_one : planes_two) + 8 * i;
    const int64_t token = row / heads;
    AttnChunk<float> c;
    attn_load(c, (const float *)s.p + token * s.n + (row - token * heads) * s.h, 8 * (int)(i % (DP / 8)), width, s.wide);
    const AttnFrag<3> f = attn_frag(c);
#pragma unroll
    for (int t = 0; t < 3; ++t)
        *(pccnn_u32x4 *)(to + t * tokens * heads * DP) = __builtin_bit_cast(pccnn_u32x4, f.t[t]);
}

// ------------------------------------------------------------------------------------------------- forward

// The running maximum is only raised when a tile exceeds it by more than this many powers of two: P then stays below
// 2^8 in f32 and bf16 (exponents to spare in both), and the accumulators are rarely scaled.
constexpr float kSlack = 8.0f;
// The maximum of a tile with a live key is never below this.  A maximum drops NaN, so without it a row whose scores are all
// NaN would look like one without keys; with it a running maximum of minus infinity means that no key was live, nothing else.
constexpr float kLowest = -FLT_MAX;

// L of a row.  A row with live keys whose sum is not positive has scores that are all NaN or minus infinity: no softmax.
__device__ __forceinline__ float log_sum(float top, float sum)
{
    if (top == -INFINITY) return -INFINITY;
    return sum > 0.0f ? top * (1.0f / kLog2e) + logf(sum) : NAN;
}

// PTERMS: the terms that probabilities are carried in, as many as the values' in f32.  In bf16 one, since a second costs what
// the large cases have least of (34123 x 100000 keys 6.8 -> 9.2 ms, 8 x 256 x 100000 555 -> 740 us); but two where a cloud has at
// most 32 rows (ATTN_FEW), one wavefront's, which wait for memory: one row over 16 x 4096 keys 32.5 -> 33.5 us, over 10^6 keys
// 110 and 110, 8 x 32 rows over 20000 keys 49 -> 51, 200 x 20 over 500 28 -> 30.  The result then has its own rounding alone
// (0.0017 of it in the 2-norm), else the probabilities' too (0.0023).
template <typename T, int DP, bool DIRECT, int PTERMS>
__global__ __launch_bounds__(kThreads) void attention_fwd_kernel(AttnArgs a)
{
    constexpr int TERMS = AttnTerms<T>::value;
    typedef Feeder<T, DP, DIRECT, false> Feed;
    typedef typename Feed::Tile Tile;
    constexpr int ROWS = Feed::ROWS, STEPS = DP / 16, BLOCKS = DP / 32;
    extern __shared__ __align__(16) uint16_t lds[];
    const int64_t block = pccnn_xcd_block(blockIdx.x, gridDim.x, a.run);
    if (block >= a.blocks) return;
    const AttnBlock b(a, block, a.k_starts);
    if (b.tile * kOwn >= b.rows) return;
    const int lane = threadIdx.x % PCCNN_WAVE, wave = threadIdx.x / PCCNN_WAVE, half = lane >> 5;
    const int row = b.tile * kOwn + wave * 32 + (lane & 31);
    const bool working = b.tile * kOwn + wave * 32 < b.rows;         // any row of this wavefront exists
    const int64_t k_at = b.k0 * a.one.n + b.head * a.one.h, v_at = b.k0 * a.two.n + b.head * a.two.h;

    int key = (int)min((int64_t)b.split * a.per_split * ROWS, (int64_t)b.keys);
    const int end = (int)min((int64_t)b.keys, key + (int64_t)a.per_split * ROWS);
    Feed k, v;
    uint64_t live = 0;
    uint8_t flag = 0;
    k.start(a.one, k_at, 1, key);
    v.start(a.two, v_at, 1, key);
    if (key < end) {
        flag = key_flag(a, b, key, lane);
        live = live_keys(a, b, key, flag, ROWS);
        k.fetch(a.one, k_at, 1, key, b.keys, live, a.mask != nullptr, a.width, Tile{lds});
        v.fetch(a.two, v_at, 1, key, b.keys, live, a.mask != nullptr, a.width, Tile{lds + Tile::ELEMENTS});
        flag = key_flag(a, b, key + ROWS, lane);
    }
    AttnFrag<TERMS> q[DP / 16];
    own_side<T, DP>(q, a.q, row < b.rows ? b.query(a, row) * a.q_n + b.head_of(a, row) * a.q_h : 0, row < b.rows, half,
                    a.width, a.wide_q);
    pccnn_f32x16 acc[DP / 32];
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt) clear(acc[dt]);
    float top = -INFINITY, sums[2] = {0.0f, 0.0f};                   // of the lane's row; the sum over the lane's keys only
    const float c2 = a.scale * kLog2e;

    // One tile: `here` holds it, `there` is where the next one goes.  That the two do not overlap is what lets the operands'
    // reads go on while the next tile is on its way.
    auto walk = [&](uint16_t *__restrict__ here, uint16_t *__restrict__ there, const uint64_t now) {
        const Tile tile_k = {here}, tile_v = {here + Tile::ELEMENTS}, next_k = {there}, next_v = {there + Tile::ELEMENTS};
        if (key + ROWS < end) {
            live = live_keys(a, b, key + ROWS, flag, ROWS);
            k.fetch(a.one, k_at, 1, key + ROWS, b.keys, live, a.mask != nullptr, a.width, next_k);
            v.fetch(a.two, v_at, 1, key + ROWS, b.keys, live, a.mask != nullptr, a.width, next_v);
            flag = key_flag(a, b, key + 2 * ROWS, lane);
        }
        if (!working || now == 0) return;
        pccnn_f32x16 s[ROWS / 32];
#pragma unroll
        for (int t = 0; t < ROWS / 32; ++t) clear(s[t]);
        AttnAhead<TERMS> ahead;
        auto key_rows = [&](int i) { return tile_k.rows(32 * (i / STEPS) + (lane & 31), 2 * (i % STEPS) + half); };
        ahead.template prime<ROWS / 32 * STEPS>(key_rows);
        ahead.template run<ROWS / 32 * STEPS>(key_rows, [&](int i, const AttnFrag<TERMS> &f) {
            attn_mma(s[i / STEPS], f, q[i % STEPS]);
        });
        auto value_columns = [&](int i) { return tile_v.columns(16 * (i / BLOCKS), 32 * (i % BLOCKS), lane); };
        ahead.template prime<ROWS / 16 * BLOCKS>(value_columns);
        if (now != first_bits(ROWS, ROWS))
#pragma unroll
            for (int t = 0; t < ROWS / 32; ++t) hide(s[t], (uint32_t)(now >> (32 * t)), half);
        float high = s[0][0];
#pragma unroll
        for (int t = 0; t < ROWS / 32; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) high = fmaxf(high, s[t][i]);
        high = fmaxf(attn_max_halves(high) * c2, kLowest);
        if (__any(high > top + kSlack)) {
            const float raised = fmaxf(top, high);
            const float shrink = __builtin_amdgcn_exp2f(top - raised);
            top = raised;
            sums[0] *= shrink;
            sums[1] *= shrink;
#pragma unroll
            for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[dt][i] *= shrink;
        }
        AttnFrag<PTERMS> p;
        ahead.template run<ROWS / 16 * BLOCKS>(value_columns, [&](int i, const AttnFrag<TERMS> &f) {
            if (i % BLOCKS == 0) {                                   // the next sixteen keys' probabilities
                pccnn_f32x16 &x = s[i / BLOCKS / 2];
                const int from = 8 * (i / BLOCKS % 2);
#pragma unroll
                for (int j = from; j < from + 8; ++j) {
                    x[j] = __builtin_amdgcn_exp2f(fmaf(x[j], c2, -top));
                    sums[j % 2] += x[j];
                }
                p = half_of<PTERMS>(x, i / BLOCKS % 2);
            }
            attn_mma(acc[i % BLOCKS], f, p);
        });
    };
    for (int stage = 0; key < end; key += ROWS, stage ^= 1) {
        uint16_t *const here = lds + stage * 2 * Tile::ELEMENTS, *const there = lds + (stage ^ 1) * 2 * Tile::ELEMENTS;
        const uint64_t now = live;
        if constexpr (DIRECT) {
            attn_landed();
        } else {
            k.put(Tile{here}, now);
            v.put(Tile{here + Tile::ELEMENTS}, now);
            __syncthreads();
        }
        walk(here, there, now);
    }
    const float sum = pccnn_add_row_xor32(sums[0] + sums[1]);
    if (row >= b.rows) return;
    const int64_t token = b.query(a, row) * a.heads + b.head_of(a, row);
    if (a.splits > 1) {
        const int64_t at = (int64_t)b.split * a.m * a.heads + token;
        const int padded = (a.width + 3) / 4 * 4;
        write_column<float, DP>(a.part + at * padded, acc, 1.0f, half, padded);
        if (half == 0) a.part_ml[at] = make_float2(top, sum);
    } else {
        const bool none = top == -INFINITY;                          // no live key at all: zeros
        write_column<T, DP>((T *)a.out + token * a.width, acc, none ? 0.0f : 1.0f / sum, half, a.width);
        if (a.lse != nullptr && half == 0) a.lse[token] = log_sum(top, sum);
    }
}

// Joins the parts of a forward pass that was split over the keys: THREADS threads to a (query, head), LANES of them side by
// side over its features (four each), the groups over the parts, added up in a fixed order.  8 results in 521 parts take
// 10 us (three dependent reads of what other XCDs wrote), 16384 results in 22 parts 25 us = 3.9 TB/s.
template <typename T, int THREADS, int BLOCK>
__global__ __launch_bounds__(BLOCK) void attention_join_kernel(AttnArgs a, int lanes)
{
    __shared__ float sums[BLOCK][5];
    const int mine = threadIdx.x % THREADS, first = threadIdx.x - mine;
    const int64_t tokens = a.m * a.heads, token = (int64_t)blockIdx.x * (BLOCK / THREADS) + threadIdx.x / THREADS;
    const int group = mine / lanes, groups = THREADS / lanes, col = mine % lanes * 4;
    float value[4] = {0.0f, 0.0f, 0.0f, 0.0f}, sum = 0.0f, top = -INFINITY;
    if (token < tokens) {
        for (int s = mine; s < a.splits; s += THREADS) top = fmaxf(top, a.part_ml[s * tokens + token].x);
    }
    top = pccnn_wave_minmax<true>(top);
    if (THREADS > PCCNN_WAVE) {
        sums[threadIdx.x][0] = top;
        __syncthreads();
        for (int i = 0; i < THREADS; i += PCCNN_WAVE) top = fmaxf(top, sums[first + i][0]);
        __syncthreads();
    }
    const float shift = top == -INFINITY ? 0.0f : top;
    const int padded = (a.width + 3) / 4 * 4;                        // a part's rows are whole units of four
    if (token < tokens && col < padded) {
        constexpr int BATCH = THREADS > PCCNN_WAVE ? 8 : 2;          // parts whose loads are on their way together
        for (int s = group; s < a.splits; s += BATCH * groups) {
            float2 ml[BATCH];
            float4 x[BATCH];
#pragma unroll
            for (int u = 0; u < BATCH; ++u) {
                const int64_t at = min(s + u * groups, a.splits - 1) * tokens + token;
                ml[u] = a.part_ml[at];
                x[u] = *(const float4 *)(a.part + at * padded + col);
            }
#pragma unroll
            for (int u = 0; u < BATCH; ++u) {
                const float w = s + u * groups < a.splits ? __builtin_amdgcn_exp2f(ml[u].x - shift) : 0.0f;
                sum = fmaf(ml[u].y, w, sum);
                value[0] = fmaf(x[u].x, w, value[0]); value[1] = fmaf(x[u].y, w, value[1]);
                value[2] = fmaf(x[u].z, w, value[2]); value[3] = fmaf(x[u].w, w, value[3]);
            }
        }
    }
    // the groups of a wavefront first, then the wavefronts of the result
    for (int o = lanes; o < PCCNN_WAVE; o *= 2) {
#pragma unroll
        for (int i = 0; i < 4; ++i) value[i] += __shfl_xor(value[i], o);
        sum += __shfl_xor(sum, o);
    }
    if (THREADS > PCCNN_WAVE) {
        const int wave = mine / PCCNN_WAVE;
        if (mine % PCCNN_WAVE < lanes) {
#pragma unroll
            for (int i = 0; i < 4; ++i) sums[first + wave * 32 + mine % PCCNN_WAVE][i] = value[i];
            sums[first + wave * 32 + mine % PCCNN_WAVE][4] = sum;
        }
        __syncthreads();
        if (group == 0) {
#pragma unroll
            for (int w = 1; w < THREADS / PCCNN_WAVE; ++w) {
#pragma unroll
                for (int i = 0; i < 4; ++i) value[i] += sums[first + w * 32 + mine][i];
                sum += sums[first + w * 32 + mine][4];
            }
        }
    }
    if (group != 0 || token >= tokens) return;
    const bool none = top == -INFINITY;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float one[1] = {none ? 0.0f : value[i] / sum};
        if (col + i < a.width) pccnn_store<1>((T *)a.out + token * a.width + col + i, one);
    }
    if (a.lse != nullptr && col == 0) a.lse[token] = log_sum(top, sum);
}

// ------------------------------------------------------------------------------------------------- backward

// What the kernel of dk and dv needs of a row, for an f32 call that wants no dq (whose kernel leaves it on the way): D = dO . O,
// and L in units of log 2 (+inf for a row without keys: every P is zero).  Two lanes to a row, which add in the order of
// the halves of a wavefront there: the same bits.
__global__ __launch_bounds__(kThreads) void attention_rows_kernel(AttnArgs a)
{
    const int64_t token = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / 2;
    const bool live = token < a.m * a.heads;
    const int64_t query = token / a.heads;
    const int head = (int)(token - query * a.heads);
    float delta = 0.0f;
    if (live)
        for (int col = 8 * (threadIdx.x % 2); col < a.width; col += 16) {
            AttnChunk<float> o, d;
            attn_load(o, (const float *)a.o + token * a.width, col, a.width, a.wide_o);
            attn_load(d, (const float *)a.g + query * a.g_n + head * a.g_h, col, a.width, a.wide_g);
#pragma unroll
            for (int i = 0; i < 8; ++i) delta = fmaf(attn_value(o, i), attn_value(d, i), delta);
        }
    delta = pccnn_group_sum<2>(delta);
    if (live && threadIdx.x % 2 == 0) {
        const int64_t at = head / a.group * (a.m * a.group) + query * a.group + head % a.group;
        const float lse = a.lse[token];
        a.shift[at] = lse == -INFINITY ? INFINITY : lse * kLog2e;
        a.delta[at] = lse == -INFINITY ? 0.0f : delta;
    }
}

template <typename T, int DP, bool DIRECT>
__global__ __launch_bounds__(kThreads) void attention_dq_kernel(AttnArgs a)
{
    constexpr int TERMS = AttnTerms<T>::value;
    typedef Feeder<T, DP, DIRECT, false> Feed;
    typedef typename Feed::Tile Tile;
    constexpr int ROWS = Feed::ROWS, STEPS = DP / 16, BLOCKS = DP / 32;
    extern __shared__ __align__(16) uint16_t lds[];
    const int64_t block = pccnn_xcd_block(blockIdx.x, gridDim.x, a.run);
    if (block >= a.blocks) return;
    const AttnBlock b(a, block, a.k_starts);
    if (b.tile * kOwn >= b.rows) return;
    const bool one_tile = TERMS == 1 && b.keys <= ROWS;              // D is formed from the probabilities (below)
    const bool wanted = a.out != nullptr;                            // else the rows' statistics alone
    if (!wanted && b.split != 0) return;
    const int lane = threadIdx.x % PCCNN_WAVE, wave = threadIdx.x / PCCNN_WAVE, half = lane >> 5;
    const int row = b.tile * kOwn + wave * 32 + (lane & 31);
    const bool working = b.tile * kOwn + wave * 32 < b.rows;
    const int64_t k_at = b.k0 * a.one.n + b.head * a.one.h, v_at = b.k0 * a.two.n + b.head * a.two.h;

    int key = (int)min((int64_t)b.split * a.per_split * ROWS, (int64_t)b.keys);
    const int end = (int)min((int64_t)b.keys, key + (int64_t)a.per_split * ROWS);
    Feed k, v;
    uint64_t live = 0;
    uint8_t flag = 0;
    k.start(a.one, k_at, 1, key);
    v.start(a.two, v_at, 1, key);
    if (key < end && (wanted || one_tile)) {
        flag = key_flag(a, b, key, lane);
        live = live_keys(a, b, key, flag, ROWS);
        k.fetch(a.one, k_at, 1, key, b.keys, live, a.mask != nullptr, a.width, Tile{lds});
        v.fetch(a.two, v_at, 1, key, b.keys, live, a.mask != nullptr, a.width, Tile{lds + Tile::ELEMENTS});
        flag = key_flag(a, b, key + ROWS, lane);
    }
    const bool real = row < b.rows;
    const int64_t query = b.query(a, real ? row : 0);
    const int head = b.head_of(a, real ? row : 0);
    AttnFrag<TERMS> q[DP / 16], g[DP / 16];
    own_side<T, DP>(q, a.q, query * a.q_n + head * a.q_h, real, half, a.width, a.wide_q);
    own_side<T, DP>(g, a.g, query * a.g_n + head * a.g_h, real, half, a.width, a.wide_g);
    // D = dO . O and L of the row, left for the other kernel by the first part
    const int64_t token = query * a.heads + head;
    float delta = 0.0f;
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) {
        AttnChunk<T> o, d;
        attn_clear(o);
        attn_clear(d);
        if (real) {
            attn_load(o, (const T *)a.o + token * a.width, 16 * kk + 8 * half, a.width, a.wide_o);
            attn_load(d, (const T *)a.g + query * a.g_n + head * a.g_h, 16 * kk + 8 * half, a.width, a.wide_g);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) delta = fmaf(attn_value(o, i), attn_value(d, i), delta);
    }
    delta = pccnn_add_row_xor32(delta);
    const float lse = real ? a.lse[token] : -INFINITY;
    const float shift = lse == -INFINITY ? INFINITY : lse * kLog2e;  // a row without keys: every P is zero
    if (lse == -INFINITY) delta = 0.0f;
    const float c2 = a.scale * kLog2e;
    // S and dP of 32 keys of a tile
    auto both = [&](const Tile &tile_k, const Tile &tile_v, int t, pccnn_f32x16 &s, pccnn_f32x16 &dp) {
        clear(s);
        clear(dp);
        AttnAhead<TERMS> ahead;
        auto rows = [&](int i) { return (i < STEPS ? tile_k : tile_v).rows(32 * t + (lane & 31), 2 * (i % STEPS) + half); };
        ahead.template prime<2 * STEPS>(rows);
        ahead.template run<2 * STEPS>(rows, [&](int i, const AttnFrag<TERMS> &f) {
            if (i < STEPS)
                attn_mma(s, f, q[i]);
            else
                attn_mma(dp, f, g[i - STEPS]);
        });
    };
    // Waits for a tile that was fetched.
    auto land = [&](uint16_t *here, const uint64_t now) {
        if constexpr (DIRECT) {
            attn_landed();
        } else {
            k.put(Tile{here}, now);
            v.put(Tile{here + Tile::ELEMENTS}, now);
            __syncthreads();
        }
    };
    // bf16: O is rounded, and D of a rounded O is off by as much of dO . O.  Among few keys that is most of dP - D (two keys: dq and
    // dk off by 0.0044 in the 2-norm where their own rounding is 0.0017), so where a cloud's keys are one tile D is formed as
    // sum P dP over it, whose products are done twice then (16 x 4096 rows over 48 keys, 8 heads of 64: dq 83 -> 87 us, all
    // gradients 118 -> 121; over 64 keys, 4 heads of 32: 27 -> 29 and 47 -> 49, keys' and values' alone 31 -> 43).
    bool landed = false;
    if (one_tile && key < end) {
        land(lds, live);
        landed = true;
        if (working) {
            float sum = 0.0f, dot = 0.0f;
#pragma unroll 1
            for (int t = 0; t < ROWS / 32; ++t) {
                pccnn_f32x16 s, dp;
                both(Tile{lds}, Tile{lds + Tile::ELEMENTS}, t, s, dp);
                hide(s, (uint32_t)(live >> (32 * t)), half);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float p = __builtin_amdgcn_exp2f(fmaf(s[i], c2, -shift));
                    sum += p;
                    dot = fmaf(p, dp[i], dot);
                }
            }
            sum = pccnn_add_row_xor32(sum);
            dot = pccnn_add_row_xor32(dot);
            if (sum > 0.0f) delta = dot / sum;
        }
    }
    if (real && half == 0 && b.split == 0) {
        a.shift[b.stat(a, row)] = shift;
        a.delta[b.stat(a, row)] = delta;
    }
    if (!wanted) return;
    pccnn_f32x16 acc[DP / 32];
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt) clear(acc[dt]);

    // One tile: `here` holds it, `there` is where the next one goes.  That the two do not overlap is what lets the operands'
    // reads go on while the next tile is on its way.
    auto walk = [&](uint16_t *__restrict__ here, uint16_t *__restrict__ there, const uint64_t now) {
        const Tile tile_k = {here}, tile_v = {here + Tile::ELEMENTS}, next_k = {there}, next_v = {there + Tile::ELEMENTS};
        if (key + ROWS < end) {
            live = live_keys(a, b, key + ROWS, flag, ROWS);
            k.fetch(a.one, k_at, 1, key + ROWS, b.keys, live, a.mask != nullptr, a.width, next_k);
            v.fetch(a.two, v_at, 1, key + ROWS, b.keys, live, a.mask != nullptr, a.width, next_v);
            flag = key_flag(a, b, key + 2 * ROWS, lane);
        }
        if (!working || now == 0) return;
#pragma unroll
        for (int t = 0; t < ROWS / 32; ++t) {
            pccnn_f32x16 s, dp;
            both(tile_k, tile_v, t, s, dp);
            AttnAhead<TERMS> ahead;
            auto columns = [&](int i) { return tile_k.columns(32 * t + 16 * (i / BLOCKS), 32 * (i % BLOCKS), lane); };
            ahead.template prime<2 * BLOCKS>(columns);
            if (now != first_bits(ROWS, ROWS)) hide(s, (uint32_t)(now >> (32 * t)), half);
            AttnFrag<TERMS> ds;
            ahead.template run<2 * BLOCKS>(columns, [&](int i, const AttnFrag<TERMS> &f) {
                if (i % BLOCKS == 0) {
                    const int from = 8 * (i / BLOCKS);
#pragma unroll
                    for (int j = from; j < from + 8; ++j)
                        s[j] = __builtin_amdgcn_exp2f(fmaf(s[j], c2, -shift)) * (dp[j] - delta);
                    ds = half_of<TERMS>(s, i / BLOCKS);
                }
                attn_mma(acc[i % BLOCKS], f, ds);
            });
        }
    };
    for (int stage = 0; key < end; key += ROWS, stage ^= 1) {
        uint16_t *const here = lds + stage * 2 * Tile::ELEMENTS, *const there = lds + (stage ^ 1) * 2 * Tile::ELEMENTS;
        const uint64_t now = live;
        if (!landed) land(here, now);
        landed = false;
        walk(here, there, now);
    }
    if (!real) return;
    if (shift == INFINITY) {                                         // whatever its gradient holds (0 times NaN)
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt) clear(acc[dt]);
    }
    if (a.splits > 1)
        write_column<float, DP>(a.part + ((int64_t)b.split * a.m * a.heads + token) * a.width, acc, a.scale, half, a.width);
    else
        write_column<T, DP>((T *)a.out + token * a.width, acc, a.scale, half, a.width);
}

template <typename T, int DP, bool DIRECT>
__global__ __launch_bounds__(kThreads) void attention_dkv_kernel(AttnArgs a)
{
    constexpr int TERMS = AttnTerms<T>::value;
    typedef Feeder<T, DP, DIRECT, true> Feed;
    typedef typename Feed::Tile Tile;
    constexpr int ROWS = Feed::ROWS, STEPS = DP / 16, BLOCKS = DP / 32;
    extern __shared__ __align__(16) uint16_t lds[];
    float *const stats = (float *)(lds + 4 * Tile::ELEMENTS);        // [stage][shift, delta][64]
    const int64_t block = pccnn_xcd_block(blockIdx.x, gridDim.x, a.run);
    if (block >= a.blocks) return;
    const AttnBlock b(a, block, a.q_starts);
    if (b.tile * kOwn >= b.keys) return;
    const int lane = threadIdx.x % PCCNN_WAVE, wave = threadIdx.x / PCCNN_WAVE, half = lane >> 5;
    const int key = b.tile * kOwn + wave * 32 + (lane & 31);
    const bool working = b.tile * kOwn + wave * 32 < b.keys;
    const bool live = key < b.keys && (a.mask == nullptr || a.mask[b.k0 + key] != 0);
    const int64_t q_at = b.q0 * a.one.n + b.head * a.group * a.one.h, g_at = b.q0 * a.two.n + b.head * a.group * a.two.h;

    int row = (int)min((int64_t)b.split * a.per_split * ROWS, (int64_t)b.rows);
    const int end = (int)min((int64_t)b.rows, row + (int64_t)a.per_split * ROWS);
    Feeder<T, DP, DIRECT, true, true> q;
    Feed g;
    q.start(a.one, q_at, a.group, row);
    g.start(a.two, g_at, a.group, row);
    // shifts and deltas of the tile's rows, one wavefront each; they pass through a register, since LDS that the compiler
    // knows to be filled behind its back would make it wait for all that is on its way
    float stat = 0.0f;
    auto fetch_stats = [&](int from) {
        if (wave < 2) {
            stat = wave == 0 ? INFINITY : 0.0f;
            if (from + lane < b.rows) stat = (wave == 0 ? a.shift : a.delta)[b.stat(a, from + lane)];
        }
    };
    if (row < end) {
        const uint64_t bits = first_bits(b.rows - row, ROWS);
        q.fetch(a.one, q_at, a.group, row, b.rows, bits, false, a.width, Tile{lds});
        g.fetch(a.two, g_at, a.group, row, b.rows, bits, false, a.width, Tile{lds + Tile::ELEMENTS});
        fetch_stats(row);
    }
    AttnFrag<TERMS> k[DP / 16], v[DP / 16];
    own_side<T, DP>(k, a.k, (b.k0 + key) * a.k_n + b.head * a.k_h, live, half, a.width, a.wide_k);
    own_side<T, DP>(v, a.v, (b.k0 + key) * a.v_n + b.head * a.v_h, live, half, a.width, a.wide_v);
    pccnn_f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt) {
        clear(dk[dt]);
        clear(dv[dt]);
    }
    const float c2 = a.scale * kLog2e;
    auto walk = [&](uint16_t *__restrict__ here, uint16_t *__restrict__ there, const float *__restrict__ stat_here) {
        const Tile tile_q = {here}, tile_g = {here + Tile::ELEMENTS}, next_q = {there}, next_g = {there + Tile::ELEMENTS};
        if (row + ROWS < end) {
            const uint64_t bits = first_bits(b.rows - row - ROWS, ROWS);
            fetch_stats(row + ROWS);
            q.fetch(a.one, q_at, a.group, row + ROWS, b.rows, bits, false, a.width, next_q);
            g.fetch(a.two, g_at, a.group, row + ROWS, b.rows, bits, false, a.width, next_g);
        }
        if (!working) return;
#pragma unroll
        for (int t = 0; t < ROWS / 32; ++t) {
            pccnn_f32x16 s, dp;
            clear(s);
            clear(dp);
            AttnAhead<TERMS> ahead;
            auto rows = [&](int i) { return (i < STEPS ? tile_q : tile_g).rows(32 * t + (lane & 31), 2 * (i % STEPS) + half); };
            ahead.template prime<2 * STEPS>(rows);
            ahead.template run<2 * STEPS>(rows, [&](int i, const AttnFrag<TERMS> &f) {
                if (i < STEPS)
                    attn_mma(s, f, k[i]);
                else
                    attn_mma(dp, f, v[i - STEPS]);
            });
            // sixteen rows at a time: first the output gradients' columns (dv), then the queries' (dk)
            auto columns = [&](int i) {
                return (i / BLOCKS % 2 == 0 ? tile_g : tile_q).columns(32 * t + 16 * (i / BLOCKS / 2), 32 * (i % BLOCKS), lane);
            };
            ahead.template prime<4 * BLOCKS>(columns);
            AttnFrag<TERMS> p, ds;
            ahead.template run<4 * BLOCKS>(columns, [&](int i, const AttnFrag<TERMS> &f) {
                if (i % (2 * BLOCKS) == 0) {
                    const int h = i / BLOCKS / 2;
#pragma unroll
                    for (int n = 2 * h; n < 2 * h + 2; ++n) {
                        const float4 shift = *(const float4 *)(stat_here + 32 * t + 8 * n + 4 * half);
                        const float4 delta = *(const float4 *)(stat_here + 64 + 32 * t + 8 * n + 4 * half);
                        const float sh[4] = {shift.x, shift.y, shift.z, shift.w}, de[4] = {delta.x, delta.y, delta.z, delta.w};
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            s[4 * n + j] = __builtin_amdgcn_exp2f(fmaf(s[4 * n + j], c2, -sh[j]));
                            dp[4 * n + j] = s[4 * n + j] * (dp[4 * n + j] - de[j]);
                        }
                    }
                    p = half_of<TERMS>(s, h);
                    ds = half_of<TERMS>(dp, h);
                }
                if (i / BLOCKS % 2 == 0)
                    attn_mma(dv[i % BLOCKS], f, p);
                else
                    attn_mma(dk[i % BLOCKS], f, ds);
            });
        }
    };
    for (int stage = 0; row < end; row += ROWS, stage ^= 1) {
        uint16_t *const here = lds + stage * 2 * Tile::ELEMENTS, *const there = lds + (stage ^ 1) * 2 * Tile::ELEMENTS;
        if constexpr (!DIRECT) {
            const uint64_t bits = first_bits(b.rows - row, ROWS);
            q.put(Tile{here}, bits);
            g.put(Tile{here + Tile::ELEMENTS}, bits);
        }
        if (wave < 2) stats[(stage * 2 + wave) * 64 + lane] = stat;
        attn_landed();
        walk(here, there, stats + stage * 128);
    }
    if (key >= b.keys) return;
    if (!live) {
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt) {
            clear(dk[dt]);
            clear(dv[dt]);
        }
    }
    const int64_t at = (b.k0 + key) * a.key_heads + b.head;
    if (a.splits > 1) {
        const int64_t part = ((int64_t)b.split * a.n * a.key_heads + at) * a.width;
        write_column<float, DP>(a.part + part, dk, a.scale, half, a.width);
        write_column<float, DP>(a.part_v + part, dv, 1.0f, half, a.width);
    } else {
        write_column<T, DP>((T *)a.d_k + at * a.width, dk, a.scale, half, a.width);
        write_column<T, DP>((T *)a.d_v + at * a.width, dv, 1.0f, half, a.width);
    }
}

// Sum of the parts of one or two gradients (blockIdx.y), in order; VEC values per thread (4 when the count is a multiple
// of 4).
template <typename T, int VEC>
__global__ __launch_bounds__(kThreads) void attention_sum_kernel(const float *__restrict__ part_one,
                                                                const float *__restrict__ part_two, int splits,
                                                                int64_t count, T *__restrict__ one, T *__restrict__ two)
{
    const int64_t i = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * VEC;
    if (i >= count) return;
    const float *part = blockIdx.y == 0 ? part_one : part_two;
    float sum[VEC], x[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) sum[j] = 0.0f;
#pragma unroll 4
    for (int s = 0; s < splits; ++s) {
        pccnn_load<VEC>(part + s * count + i, x);
#pragma unroll
        for (int j = 0; j < VEC; ++j) sum[j] += x[j];
    }
    pccnn_store<VEC>((blockIdx.y == 0 ? one : two) + i, sum);
}

// ------------------------------------------------------------------------------------------------- host side

// Everything but the pointers, which a caller who asks for the workspace's size need not have yet.
int attn_check_sizes(const char *name, const pccnn_attention *p)
{
    PCCNN_REQUIRE(p != nullptr, PCCNN_ERR_INVALID, "%s: null pointer", name);
    PCCNN_REQUIRE(pccnn_type_ok(p->type), PCCNN_ERR_UNSUPPORTED, "%s: element type %d (f32 and bf16 only)", name, p->type);
    PCCNN_REQUIRE(p->m >= 0 && p->n >= 0 && p->clouds >= 0 && p->max_queries >= 0 && p->max_keys >= 0 &&
                      p->max_queries <= p->m && p->max_keys <= p->n,
                  PCCNN_ERR_INVALID, "%s: m=%lld, n=%lld, %d clouds of up to %lld queries and %lld keys", name,
                  (long long)p->m, (long long)p->n, p->clouds, (long long)p->max_queries, (long long)p->max_keys);
    PCCNN_REQUIRE(p->heads >= 1 && p->key_heads >= 1 && p->heads % p->key_heads == 0 && p->width >= 1, PCCNN_ERR_INVALID,
                  "%s: %d heads, %d key heads, width %d (heads: a multiple of key heads)", name, p->heads, p->key_heads,
                  p->width);
    PCCNN_REQUIRE(p->width <= kMaxWidth, PCCNN_ERR_UNSUPPORTED, "%s: head width %d (up to %d)", name, p->width, kMaxWidth);
    PCCNN_REQUIRE(p->m <= INT32_MAX && p->n <= INT32_MAX - kOwn &&
                      p->max_queries * (p->heads / p->key_heads) <= (int64_t)INT32_MAX - 4 * kOwn,
                  PCCNN_ERR_UNSUPPORTED, "%s: m=%lld, n=%lld: starts are 32-bit", name, (long long)p->m, (long long)p->n);
    PCCNN_REQUIRE(p->scale > 0.0f && p->scale <= 3.0e38f, PCCNN_ERR_INVALID, "%s: scale=%g (positive and finite)", name,
                  (double)p->scale);
    PCCNN_REQUIRE(p->m * p->heads <= kMostTokens && p->n * p->key_heads <= kMostTokens, PCCNN_ERR_UNSUPPORTED,
                  "%s: %lld queries of %d heads, %lld keys of %d (up to 2^32 of both)", name, (long long)p->m, p->heads,
                  (long long)p->n, p->key_heads);
    const int64_t strides[] = {p->q_stride_n, p->q_stride_h, p->k_stride_n, p->k_stride_h, p->v_stride_n, p->v_stride_h};
    for (int64_t s : strides)
        PCCNN_REQUIRE(s >= 0, PCCNN_ERR_INVALID, "%s: a stride of %lld elements", name, (long long)s);
    return PCCNN_OK;
}
int attn_check(const char *name, const pccnn_attention *p)
{
    const int rc = attn_check_sizes(name, p);
    if (rc != PCCNN_OK) return rc;
    PCCNN_REQUIRE(p->m == 0 || p->clouds == 0 || (p->queries && p->query_starts && p->key_starts), PCCNN_ERR_INVALID,
                  "%s: null pointer", name);
    PCCNN_REQUIRE(p->n == 0 || p->clouds == 0 || (p->keys && p->values && p->query_starts && p->key_starts),
                  PCCNN_ERR_INVALID, "%s: null pointer", name);
    return PCCNN_OK;
}

int attn_wide(const void *p, int64_t stride_n, int64_t stride_h, int type, int width)
{
    for (int count = 8; count >= 4; count /= 2) {
        const int bytes = std::min(16, count * pccnn_type_bytes(type));
        if (width % count == 0 && pccnn_rows_aligned(p, stride_n, type, bytes) &&
            pccnn_rows_aligned(p, stride_h, type, bytes))
            return count / 4;
    }
    return 0;
}

AttnArgs attn_args(const pccnn_attention *p)
{
    AttnArgs a = {};
    a.q = p->queries; a.k = p->keys; a.v = p->values;
    a.q_n = p->q_stride_n; a.q_h = p->q_stride_h;
    a.k_n = p->k_stride_n; a.k_h = p->k_stride_h;
    a.v_n = p->v_stride_n; a.v_h = p->v_stride_h;
    a.q_starts = p->query_starts; a.k_starts = p->key_starts; a.mask = p->key_mask;
    a.m = p->m; a.n = p->n;
    a.clouds = p->clouds; a.heads = p->heads; a.key_heads = p->key_heads; a.group = p->heads / p->key_heads;
    a.width = p->width; a.scale = p->scale;
    a.wide_q = attn_wide(a.q, a.q_n, a.q_h, p->type, a.width);
    a.wide_k = attn_wide(a.k, a.k_n, a.k_h, p->type, a.width);
    a.wide_v = attn_wide(a.v, a.v_n, a.v_h, p->type, a.width);
    a.one = a.two = AttnStream{};
    a.splits = 1;
    return a;
}

// Whether a tile's rows, strides apart, are within 32-bit offsets in bytes of its first one.
bool attn_reachable(int64_t stride_n, int64_t stride_h, int group)
{
    return std::max(stride_n, stride_h) < (1ll << 30) &&
           64 * stride_n + std::max<int64_t>(64, group) * stride_h + kMaxWidth < (1ll << 30);
}
// Whether the walked side, of `heads` heads, goes to LDS without passing registers.  bf16: where rows are whole 16-byte units
// with 32-bit offsets within a tile.  f32: where it is worth turning into planes of terms first, that is where each cloud has
// several own tiles (`own`: rows of all clouds) to walk it, and the planes' tiles have such offsets.
bool attn_direct(const AttnArgs &a, int type, const AttnStream &one, const AttnStream &two, int heads, int64_t own)
{
    const int64_t padded = (a.width + 31) / 32 * 32;
    if (type == PCCNN_TYPE_F32)
        return own >= (int64_t)kPlanesFrom * kOwn * a.clouds && attn_reachable(heads * padded, padded, a.group);
    return one.wide == 2 && two.wide == 2 && attn_reachable(std::max(one.n, two.n), std::max(one.h, two.h), a.group);
}

// Calls f(type, padded width) for the instantiation that serves this type and head width.
template <typename F> auto attn_dispatch(int type, int width, F f)
{
    auto by_width = [&](auto zero) {
        if (width <= 32) return f(zero, std::integral_constant<int, 32>());
        if (width <= 64) return f(zero, std::integral_constant<int, 64>());
        if (width <= 96) return f(zero, std::integral_constant<int, 96>());
        return f(zero, std::integral_constant<int, 128>());
    };
    return type == PCCNN_TYPE_F32 ? by_width(0.0f) : by_width((uint16_t)0);
}

// Workgroups of a kernel that are on the chip at once.
template <typename KERNEL> int attn_slots(KERNEL kernel, size_t lds)
{
    int device = 0, cus = 0, per_cu = 0;
    if (hipGetDevice(&device) != hipSuccess ||
        hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess ||
        hipOccupancyMaxActiveBlocksPerMultiprocessor(&per_cu, (const void *)kernel, kThreads, lds) != hipSuccess ||
        cus < 1 || per_cu < 1) {
        (void)hipGetLastError();
        return 512;                          // no device to ask: two per CU
    }
    return cus * per_cu;
}
enum AttnPass { ATTN_FORWARD, ATTN_FEW, ATTN_QUERIES, ATTN_KEYS };

// The kernel of a pass, its LDS and the workgroups that are resident at once (asked once).
struct AttnKernel {
    void (*run)(AttnArgs);
    size_t lds;
    int slots, rows;
    bool direct;
};
template <typename T, int DP, bool DIRECT, AttnPass PASS> AttnKernel attn_kernel()
{
    AttnKernel k;
    constexpr int TERMS = AttnTerms<T>::value;
    if constexpr (PASS == ATTN_FORWARD) k.run = attention_fwd_kernel<T, DP, DIRECT, TERMS>;
    if constexpr (PASS == ATTN_FEW) k.run = attention_fwd_kernel<T, DP, DIRECT, TERMS == 1 ? 2 : TERMS>;
    if constexpr (PASS == ATTN_QUERIES) k.run = attention_dq_kernel<T, DP, DIRECT>;
    if constexpr (PASS == ATTN_KEYS) k.run = attention_dkv_kernel<T, DP, DIRECT>;
    k.rows = attn_tile_rows<T, DP>();
    k.direct = DIRECT;
    // two tiles of two tensors, and the backward rows' statistics
    k.lds = 4 * 2 * (size_t)AttnTile<AttnTerms<T>::value, attn_tile_rows<T, DP>(), DP>::ELEMENTS +
            (PASS == ATTN_KEYS ? 4 * 64 * sizeof(float) : 0);
    static const int slots = attn_slots(k.run, k.lds);
    k.slots = slots;
    return k;
}
template <AttnPass PASS> AttnKernel attn_kernel_of(int type, int width, bool direct)
{
    return attn_dispatch(type, width, [&](auto zero, auto dp) -> AttnKernel {
        using T = decltype(zero);
        constexpr int DP = decltype(dp)::value;
        return direct ? attn_kernel<T, DP, true, PASS>() : attn_kernel<T, DP, false, PASS>();
    });
}

// Into how many parts the other side is cut.  More parts even out the last round of workgroups (1068 tiles on 512 places
// take three rounds where 2.1 would do) and fill the chip when there are few tiles, but each part writes its sums in f32
// and they are read again by the join.  The estimate below (microseconds) weighs the two: a tile of the other side costs a
// place its share of 900 TFLOP/s of bf16 products (six per product in f32) or of 5 TB/s, whichever is longer; parts cost
// their bytes at 4 TB/s and a launch.
void attn_plan(AttnArgs &a, const AttnKernel &kernel, int type, int products, int64_t own, int64_t own_all, int64_t other,
               int64_t other_all)
{
    const double terms = type == PCCNN_TYPE_F32 ? 6.0 : 1.0, padded = (a.width + 31) / 32 * 32.0;
    const double unit = kernel.slots * std::max(2.0 * products * kOwn * kernel.rows * padded * terms / 900e6,
                                                2.0 * kernel.rows * a.width * pccnn_type_bytes(type) / 5e6);
    const double result = (double)own_all * a.key_heads * a.width * 4 * (products == 4 ? 2 : 1);     // bytes of one part
    a.tiles = (int)std::max<int64_t>(1, pccnn_ceil_div(own, kOwn));
    const int64_t tiles = std::max<int64_t>(1, pccnn_ceil_div(other, kernel.rows));
    // workgroups that have work, and the tiles a mean one walks (clouds differ in size)
    const double mean_own = (double)own_all / a.clouds, mean_other = (double)other_all / a.clouds;
    const double groups = a.key_heads * (double)a.clouds * std::min<double>(a.tiles, std::max(1.0, mean_own / kOwn + 0.5));
    const double mean_tiles = std::min<double>((double)tiles, std::max(1.0, mean_other / kernel.rows + 0.5));
    double best = 1e300;
    for (int64_t s = 1; s <= tiles; s += s < 8 ? 1 : s / 4) {
        const int64_t per = pccnn_ceil_div(tiles, s), parts = pccnn_ceil_div(tiles, per);
        const double work = groups * (mean_tiles + 2.0 * std::min<double>((double)parts, mean_tiles / per + 1.0));
        const double rounds = std::ceil(groups * parts / kernel.slots - 0.01) * (std::min<double>((double)per, mean_tiles) + 2.0);
        const double cost = unit * std::max(rounds, work / kernel.slots + 0.5 * per) +
                            (parts > 1 ? 6.0 + 0.01 * parts + 2.0 * parts * result / 4e6 : 0.0);
        if (cost < best) {
            best = cost;
            a.per_split = (int)per;
            a.splits = (int)parts;
        }
    }
    // Workgroups that walk the same tiles on one XCD: its L2 serves them once (8 x 256 rows over 100000 keys 605 -> 560 us,
    // dk and dv 970 -> 945).  The XCDs are dealt their workgroups in turn, whatever these weigh, so where clouds differ the
    // runs are all tiles of a head and only where a cloud's heads and parts fill the eight evenly (8 uneven clouds of 8
    // heads: 216 -> 187 us, with runs of 16 242), else single workgroups.  Against single workgroups, runs of 8 and of all
    // tiles for every call, over nine uneven batches of 3 to 30 clouds, 2 to 16 heads and 32 to 128 features, 23 of 27 passes
    // are within 5 % of the best of the three; the others lose 8 to 14 % to runs of 8 or of all tiles (dk and dv of 16 clouds of
    // 4 heads and of 12 of 2 key heads, dq and dk, dv of 6 f32 clouds of 4 heads).
    const bool uneven = other * a.clouds > other_all || own * a.clouds > own_all;
    const int64_t blocks = (int64_t)a.tiles * a.splits * a.key_heads * a.clouds;
    a.run = uneven ? (a.key_heads * a.splits % PCCNN_XCDS == 0 ? a.tiles : 1) : blocks >= 4 * kernel.slots ? 16 : 8;
    a.longest_first = a.clouds > 1 && a.clouds <= PCCNN_WAVE && other * a.clouds > other_all &&
                      (double)a.tiles * a.splits * a.key_heads * a.clouds > kernel.slots;
}
// The three passes: which side is walked, by which kernel, in how many parts.
AttnKernel attn_plan_rows(AttnArgs &a, const pccnn_attention *p, bool forward)
{
    a.one = {a.k, a.k_n, a.k_h, 0, a.wide_k, a.width / 8};
    a.two = {a.v, a.v_n, a.v_h, 0, a.wide_v, a.width / 8};
    const bool direct = attn_direct(a, p->type, a.one, a.two, a.key_heads, p->m * a.group);
    const AttnKernel kernel = !forward ? attn_kernel_of<ATTN_QUERIES>(p->type, a.width, direct)
                              : p->max_queries * a.group <= 32 ? attn_kernel_of<ATTN_FEW>(p->type, a.width, direct)
                                                               : attn_kernel_of<ATTN_FORWARD>(p->type, a.width, direct);
    attn_plan(a, kernel, p->type, forward ? 2 : 3, p->max_queries * a.group, p->m * a.group, p->max_keys, p->n);
    return kernel;
}
AttnKernel attn_plan_keys(AttnArgs &a, const pccnn_attention *p, bool direct)
{
    const AttnKernel kernel = attn_kernel_of<ATTN_KEYS>(p->type, a.width, direct);
    attn_plan(a, kernel, p->type, 4, p->max_keys, p->n, p->max_queries * a.group, p->m * a.group);
    return kernel;
}
// Bytes of the two tensors' planes, when the pass works on planes.
size_t planes_bytes(const AttnArgs &a, int type, const AttnKernel &kernel, int64_t tokens, int heads)
{
    if (type != PCCNN_TYPE_F32 || !kernel.direct) return 0;
    return 2 * pccnn_align((size_t)3 * tokens * heads * ((a.width + 31) / 32 * 32) * sizeof(uint16_t));
}
// Turns the walked side into planes and lets the pass walk those.
int attn_planes(AttnArgs &a, int type, const AttnKernel &kernel, int64_t tokens, int heads, PccnnArena &arena, hipStream_t s)
{
    if (type != PCCNN_TYPE_F32 || !kernel.direct || tokens == 0) return PCCNN_OK;      // (no tokens: nothing is walked)
    return attn_dispatch(type, a.width, [&](auto, auto dp) -> int {
        constexpr int DP = decltype(dp)::value;
        const size_t count = (size_t)tokens * heads * DP;
        uint16_t *one = arena.take<uint16_t>(3 * count), *two = arena.take<uint16_t>(3 * count);
        PCCNN_REQUIRE(arena.ok(), PCCNN_ERR_WORKSPACE, "cross_attention: workspace of %zu bytes is too small", arena.size);
        const dim3 grid((unsigned)pccnn_ceil_div((int64_t)count / 8, kThreads), 2);
        attention_planes_kernel<DP><<<grid, kThreads, 0, s>>>(a.one, a.two, tokens, heads, a.width, one, two);
        PCCNN_LAUNCH_CHECK();
        a.one = {one, (int64_t)heads * DP, DP, (int64_t)count, 2, DP / 8};
        a.two = {two, (int64_t)heads * DP, DP, (int64_t)count, 2, DP / 8};
        return PCCNN_OK;
    });
}

int64_t attn_blocks(const AttnArgs &a) { return (int64_t)a.tiles * a.splits * a.key_heads * a.clouds; }

int attn_launch(const char *name, const AttnKernel &kernel, AttnArgs &a, hipStream_t s)
{
    const int64_t blocks = attn_blocks(a);
    a.blocks = blocks;
    PCCNN_REQUIRE(blocks <= INT32_MAX - PCCNN_XCDS * (int64_t)a.run, PCCNN_ERR_UNSUPPORTED, "%s: %lld workgroups", name, (long long)blocks);
    if (kernel.lds > 65536)
        PCCNN_HIP_CHECK(hipFuncSetAttribute((const void *)kernel.run, hipFuncAttributeMaxDynamicSharedMemorySize,
                                            (int)kernel.lds));
    kernel.run<<<pccnn_xcd_grid(blocks, a.run), kThreads, kernel.lds, s>>>(a);
    PCCNN_LAUNCH_CHECK();
    return PCCNN_OK;
}

size_t forward_bytes(const AttnArgs &a)
{
    if (a.splits == 1) return 0;
    const size_t tokens = (size_t)a.splits * a.m * a.heads;
    return pccnn_align(tokens * ((a.width + 3) / 4 * 4) * sizeof(float)) + pccnn_align(tokens * sizeof(float2));
}

} // namespace

extern "C" size_t pccnn_attention_workspace_bytes(const pccnn_attention *p, int backward)
{
    if (attn_check_sizes("attention_workspace_bytes", p) != PCCNN_OK || p->clouds < 1) return 256;   // (the call will refuse)
    AttnArgs a = attn_args(p);
    AttnKernel kernel = attn_plan_rows(a, p, !backward);
    size_t rows = planes_bytes(a, p->type, kernel, p->n, a.key_heads);
    if (!backward) return 256 + rows + forward_bytes(a);
    if (a.splits > 1) rows += pccnn_align((size_t)a.splits * a.m * a.heads * a.width * sizeof(float));
    size_t keys = 0;
    for (bool direct : {false, true}) {              // which one the gradient's layout allows is not known here
        kernel = attn_plan_keys(a, p, direct);
        const size_t parts = a.splits > 1
                                 ? 2 * pccnn_align((size_t)a.splits * a.n * a.key_heads * a.width * sizeof(float)) : 0;
        keys = std::max(keys, parts + planes_bytes(a, p->type, kernel, p->m, a.heads));
    }
    return 256 + 2 * pccnn_align((size_t)a.m * a.heads * sizeof(float)) + std::max(rows, keys);
}

extern "C" int pccnn_attention_forward(const pccnn_attention *p, void *out, float *lse_out, void *workspace,
                                       size_t workspace_bytes, void *stream)
{
    int rc = attn_check("cross_attention", p);
    if (rc != PCCNN_OK) return rc;
    if (p->m == 0 || p->clouds == 0) return PCCNN_OK;
    PCCNN_REQUIRE(out != nullptr, PCCNN_ERR_INVALID, "cross_attention: null pointer");
    PCCNN_REQUIRE((uintptr_t)out % 16 == 0, PCCNN_ERR_INVALID, "cross_attention: a result that is not 16-byte aligned");
    const hipStream_t s = (hipStream_t)stream;
    AttnArgs a = attn_args(p);
    a.out = out;
    a.lse = lse_out;
    const AttnKernel kernel = attn_plan_rows(a, p, true);
    PccnnArena arena(workspace, workspace_bytes);
    rc = attn_planes(a, p->type, kernel, p->n, a.key_heads, arena, s);
    if (rc != PCCNN_OK) return rc;
    if (a.splits > 1) {
        a.part = arena.take<float>((size_t)a.splits * a.m * a.heads * ((a.width + 3) / 4 * 4));
        a.part_ml = arena.take<float2>((size_t)a.splits * a.m * a.heads);
        PCCNN_REQUIRE(arena.ok(), PCCNN_ERR_WORKSPACE, "cross_attention: workspace of %zu bytes is too small",
                      workspace_bytes);
    }
    rc = attn_launch("cross_attention", kernel, a, s);
    if (rc != PCCNN_OK || a.splits == 1) return rc;
    // a wavefront to a result up to 32 parts, a workgroup of sixteen beyond
    int lanes = 1;
    while (4 * lanes < a.width) lanes *= 2;
    auto join = [&](auto zero) {
        using T = decltype(zero);
        if (a.splits <= 32)
            attention_join_kernel<T, 64, 256><<<(unsigned)pccnn_ceil_div(a.m * a.heads, 4), 256, 0, s>>>(a, lanes);
        else
            attention_join_kernel<T, 1024, 1024><<<(unsigned)(a.m * a.heads), 1024, 0, s>>>(a, lanes);
    };
    if (p->type == PCCNN_TYPE_F32)
        join(0.0f);
    else
        join((uint16_t)0);
    PCCNN_LAUNCH_CHECK();
    return PCCNN_OK;
}

extern "C" int pccnn_attention_backward(const pccnn_attention *p, const void *out, const float *lse, const void *in_grads,
                                        int64_t grads_stride_n, int64_t grads_stride_h, void *d_queries, void *d_keys,
                                        void *d_values, void *workspace, size_t workspace_bytes, void *stream)
{
    const char *name = "cross_attention_grads";
    int rc = attn_check(name, p);
    if (rc != PCCNN_OK) return rc;
    PCCNN_REQUIRE(grads_stride_n >= 0 && grads_stride_h >= 0, PCCNN_ERR_INVALID, "%s: a negative stride", name);
    PCCNN_REQUIRE((d_keys != nullptr) == (d_values != nullptr), PCCNN_ERR_INVALID,
                  "%s: the gradients of keys and values come together", name);
    if (p->clouds == 0 || (d_queries == nullptr && d_keys == nullptr)) return PCCNN_OK;
    PCCNN_REQUIRE(p->m == 0 || (out && lse && in_grads), PCCNN_ERR_INVALID, "%s: null pointer", name);
    PCCNN_REQUIRE(((uintptr_t)d_queries | (uintptr_t)d_keys | (uintptr_t)d_values) % 16 == 0, PCCNN_ERR_INVALID,
                  "%s: a result that is not 16-byte aligned", name);
    const hipStream_t s = (hipStream_t)stream;
    AttnArgs a = attn_args(p);
    a.g = in_grads;
    a.g_n = grads_stride_n;
    a.g_h = grads_stride_h;
    a.wide_g = attn_wide(a.g, a.g_n, a.g_h, p->type, a.width);
    a.wide_o = attn_wide(out, a.width, a.width, p->type, a.width);
    a.lse = (float *)lse;
    a.o = out;
    PccnnArena arena(workspace, workspace_bytes);
    auto in_workspace = [&]() -> int {
        PCCNN_REQUIRE(arena.ok(), PCCNN_ERR_WORKSPACE, "%s: workspace of %zu bytes is too small", name, workspace_bytes);
        return PCCNN_OK;
    };
    auto sum_parts = [&](const float *part_one, const float *part_two, int64_t count, void *one, void *two) {
        auto sum = [&](auto zero) {
            using T = decltype(zero);
            const unsigned tensors = two != nullptr ? 2 : 1;
            if (count % 4 == 0)
                attention_sum_kernel<T, 4><<<dim3((unsigned)pccnn_ceil_div(count, 4 * kThreads), tensors), kThreads, 0, s>>>(
                    part_one, part_two, a.splits, count, (T *)one, (T *)two);
            else
                attention_sum_kernel<T, 1><<<dim3((unsigned)pccnn_ceil_div(count, kThreads), tensors), kThreads, 0, s>>>(
                    part_one, part_two, a.splits, count, (T *)one, (T *)two);
        };
        if (p->type == PCCNN_TYPE_F32)
            sum(0.0f);
        else
            sum((uint16_t)0);
    };
    if (p->m > 0) {
        a.shift = arena.take<float>((size_t)p->m * p->heads);
        a.delta = arena.take<float>((size_t)p->m * p->heads);
        if ((rc = in_workspace()) != PCCNN_OK) return rc;
    }
    const size_t after = arena.used;
    if (d_queries != nullptr && p->m > 0) {
        const AttnKernel kernel = attn_plan_rows(a, p, false);
        const int64_t count = a.m * a.heads * a.width;
        a.out = d_queries;
        if ((rc = attn_planes(a, p->type, kernel, p->n, a.key_heads, arena, s)) != PCCNN_OK) return rc;
        if (a.splits > 1) a.part = arena.take<float>((size_t)a.splits * count);
        if ((rc = in_workspace()) != PCCNN_OK) return rc;
        rc = attn_launch(name, kernel, a, s);
        if (rc != PCCNN_OK) return rc;
        if (a.splits > 1) sum_parts(a.part, nullptr, count, d_queries, nullptr);
        PCCNN_LAUNCH_CHECK();
    }
    if (d_keys != nullptr && p->n > 0) {
        if (d_queries == nullptr && p->m > 0) {
            if (p->type == PCCNN_TYPE_F32) {
                attention_rows_kernel<<<(unsigned)pccnn_ceil_div(a.m * a.heads * 2, kThreads), kThreads, 0, s>>>(a);
                PCCNN_LAUNCH_CHECK();
            } else {                                 // (D of clouds of few keys takes their keys and values)
                const AttnKernel kernel = attn_plan_rows(a, p, false);
                a.out = nullptr;
                a.splits = 1;
                if ((rc = attn_launch(name, kernel, a, s)) != PCCNN_OK) return rc;
            }
        }
        a.one = {a.q, a.q_n, a.q_h, 0, a.wide_q, a.width / 8};
        a.two = {a.g, a.g_n, a.g_h, 0, a.wide_g, a.width / 8};
        const AttnKernel kernel = attn_plan_keys(a, p, attn_direct(a, p->type, a.one, a.two, a.heads, p->n));
        const int64_t count = a.n * a.key_heads * a.width;
        a.d_k = d_keys;
        a.d_v = d_values;
        arena.used = after;
        if ((rc = attn_planes(a, p->type, kernel, p->m, a.heads, arena, s)) != PCCNN_OK) return rc;
        if (a.splits > 1) {
            a.part = arena.take<float>((size_t)a.splits * count);
            a.part_v = arena.take<float>((size_t)a.splits * count);
        }
        if ((rc = in_workspace()) != PCCNN_OK) return rc;
        rc = attn_launch(name, kernel, a, s);
        if (rc != PCCNN_OK) return rc;
        if (a.splits > 1) sum_parts(a.part, a.part_v, count, d_keys, d_values);
        PCCNN_LAUNCH_CHECK();
    }
    return PCCNN_OK;
}
