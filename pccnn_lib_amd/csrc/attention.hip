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
#include "attention_tiles.h"

#include <algorithm>
#include <math.h>

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / PCCNN_WAVE;
constexpr int kOwn = 32 * kWaves;            // rows (forward, dq) or keys (dk, dv) of a workgroup
constexpr int kTile = 64;                    // the other side's rows in LDS at a time
constexpr int kMaxWidth = 128;
constexpr float kLog2e = 1.44269504088896341f;

struct AttnArgs {
    const void *q, *k, *v, *g;               // queries, keys, values, gradient of the output
    int64_t q_n, q_h, k_n, k_h, v_n, v_h, g_n, g_h;
    const int32_t *q_starts, *k_starts;
    const uint8_t *mask;
    int64_t m, n;
    int clouds, heads, key_heads, group, width;
    float scale;
    int wide_q, wide_k, wide_v, wide_g;
    int tiles, splits, per_split;            // own tiles per cloud and head; parts of the other side and tiles in each
    void *out;                               // forward: O; backward: dq
    float *lse, *delta;                      // [m, heads]
    void *d_k, *d_v;
    float *part, *part_v;                    // [split][rows or keys][heads][width] f32, when splits > 1
    float2 *part_ml;                         // [split][m][heads] (maximum in units of log 2, sum)
};

// The part of the problem a workgroup works on: logical block = ((cloud * key_heads + head) * splits + split) * tiles + tile.
struct AttnBlock {
    int64_t q0, k0;                          // first query and key of the cloud
    int rows, keys;                          // rows = queries * group
    int head, split, tile;
    __device__ __forceinline__ AttnBlock(const AttnArgs &a, int64_t block)
    {
        tile = (int)(block % a.tiles);
        block /= a.tiles;
        split = (int)(block % a.splits);
        block /= a.splits;
        head = (int)(block % a.key_heads);
        const int cloud = (int)(block / a.key_heads);
        // starts outside the tensors are a caller's mistake, but never an access outside them
        const int64_t q1 = min(max((int64_t)a.q_starts[cloud + 1], (int64_t)0), a.m);
        const int64_t k1 = min(max((int64_t)a.k_starts[cloud + 1], (int64_t)0), a.n);
        q0 = min(max((int64_t)a.q_starts[cloud], (int64_t)0), q1);
        k0 = min(max((int64_t)a.k_starts[cloud], (int64_t)0), k1);
        rows = (int)min((q1 - q0) * a.group, (int64_t)INT32_MAX - 2 * kOwn);
        keys = (int)(k1 - k0);
    }
    // Token (query * heads + head) of a row.
    __device__ __forceinline__ int64_t query(const AttnArgs &a, int row) const { return q0 + row / a.group; }
    __device__ __forceinline__ int head_of(const AttnArgs &a, int row) const { return head * a.group + row % a.group; }
};

// Which of the 64 keys from `key` on take part: within the cloud and not switched off.
__device__ __forceinline__ uint64_t live_keys(const AttnArgs &a, const AttnBlock &b, int key, int lane)
{
    const int mine = key + lane;
    return __ballot(mine < b.keys && (a.mask == nullptr || a.mask[b.k0 + mine] != 0));
}

// The part of a 64-row tile (DP features each) that a thread carries from memory to LDS.
template <typename T, int DP> struct Carrier {
    static constexpr int TERMS = AttnTerms<T>::value;
    static constexpr int PER_ROW = DP / 8;
    static constexpr int COUNT = kTile * PER_ROW / kThreads;
    AttnChunk<T> c[COUNT];
    // rows from `row` on of `limit`, at base + (row of the tile) * stride
    __device__ __forceinline__ void load(const T *base, int64_t stride, int row, int limit, int width, int wide)
    {
#pragma unroll
        for (int j = 0; j < COUNT; ++j) {
            const int i = threadIdx.x + j * kThreads, r = row + i / PER_ROW, col = 8 * (i % PER_ROW);
            if (r < limit)
                attn_load(c[j], base + r * stride, col, width, wide);
            else
                attn_clear(c[j]);
        }
    }
    // rows of the problem: row -> (query, head of the group)
    __device__ __forceinline__ void load_rows(const T *base, int64_t stride_n, int64_t stride_h, int row, int limit,
                                              int group, int width, int wide)
    {
#pragma unroll
        for (int j = 0; j < COUNT; ++j) {
            const int i = threadIdx.x + j * kThreads, r = row + i / PER_ROW, col = 8 * (i % PER_ROW);
            if (r < limit) {
                const int query = group == 1 ? r : r / group;
                attn_load(c[j], base + query * stride_n + (r - query * group) * stride_h, col, width, wide);
            } else {
                attn_clear(c[j]);
            }
        }
    }
    // a row whose bit is not set becomes zeros, whatever was loaded
    __device__ __forceinline__ void put(const AttnTile<TERMS, kTile, DP> &tile, uint64_t live) const
    {
#pragma unroll
        for (int j = 0; j < COUNT; ++j) {
            const int i = threadIdx.x + j * kThreads, r = i / PER_ROW, col = 8 * (i % PER_ROW);
            AttnChunk<T> chunk = c[j];
            if (!((live >> r) & 1)) attn_clear(chunk);
            tile.put(r, col, attn_frag(chunk));
        }
    }
};

// Sets scores of keys that do not take part to minus infinity (registers of C for the 32 keys from bit 0 of `live`).
__device__ __forceinline__ void hide(pccnn_f32x16 &s, uint32_t live, int half)
{
    const uint32_t mine = live >> (4 * half);
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if (!((mine >> (8 * (i / 4) + i % 4)) & 1)) s[i] = -INFINITY;
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

// ------------------------------------------------------------------------------------------------- forward

template <typename T, int DP>
__global__ __launch_bounds__(kThreads) void attention_fwd_kernel(AttnArgs a)
{
    constexpr int TERMS = AttnTerms<T>::value;
    extern __shared__ __align__(16) uint16_t lds[];
    const AttnTile<TERMS, kTile, DP> tile_k = {lds}, tile_v = {lds + TERMS * AttnTile<TERMS, kTile, DP>::PLANE};
    const AttnBlock b(a, blockIdx.x);
    if (b.tile * kOwn >= b.rows) return;
    const int lane = threadIdx.x % PCCNN_WAVE, wave = threadIdx.x / PCCNN_WAVE, half = lane >> 5;
    const int row = b.tile * kOwn + wave * 32 + (lane & 31);
    const bool working = b.tile * kOwn + wave * 32 < b.rows;         // any row of this wavefront exists
    const T *k = (const T *)a.k + b.k0 * a.k_n + b.head * a.k_h;
    const T *v = (const T *)a.v + b.k0 * a.v_n + b.head * a.v_h;

    AttnFrag<TERMS> q[DP / 16];
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) {
        AttnChunk<T> c;
        attn_clear(c);
        if (row < b.rows)
            attn_load(c, (const T *)a.q + b.query(a, row) * a.q_n + b.head_of(a, row) * a.q_h, 16 * kk + 8 * half, a.width,
                      a.wide_q);
        q[kk] = attn_frag(c);
    }
    pccnn_f32x16 acc[DP / 32];
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt) clear(acc[dt]);
    float top = -INFINITY, sum = 0.0f;                               // of the lane's row; the sum over the lane's keys only
    const float c2 = a.scale * kLog2e;

    int key = b.split * a.per_split * kTile;
    const int end = min(b.keys, key + a.per_split * kTile);
    Carrier<T, DP> next_k, next_v;
    uint64_t next_live = 0;
    if (key < end) {
        next_k.load(k, a.k_n, key, b.keys, a.width, a.wide_k);
        next_v.load(v, a.v_n, key, b.keys, a.width, a.wide_v);
        next_live = live_keys(a, b, key, lane);
    }
    for (; key < end; key += kTile) {
        const uint64_t live = next_live;
        __syncthreads();
        next_k.put(tile_k, live);
        next_v.put(tile_v, live);
        __syncthreads();
        if (key + kTile < end) {
            next_k.load(k, a.k_n, key + kTile, b.keys, a.width, a.wide_k);
            next_v.load(v, a.v_n, key + kTile, b.keys, a.width, a.wide_v);
            next_live = live_keys(a, b, key + kTile, lane);
        }
        if (!working || live == 0) continue;
        pccnn_f32x16 s[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            clear(s[t]);
#pragma unroll
            for (int kk = 0; kk < DP / 16; ++kk)
                attn_mma<TERMS>(s[t], tile_k.rows(32 * t + (lane & 31), 16 * kk + 8 * half), q[kk]);
            if (live != ~0ull) hide(s[t], (uint32_t)(live >> (32 * t)), half);
        }
        float high = s[0][0];
#pragma unroll
        for (int i = 0; i < 16; ++i) high = fmaxf(high, fmaxf(s[0][i], s[1][i]));
        high = fmaxf(top, attn_max_halves(high) * c2);
        const float shift = high == -INFINITY ? 0.0f : high;
        const float shrink = __builtin_amdgcn_exp2f(top - shift);
        top = high;
        sum *= shrink;
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[dt][i] *= shrink;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[t][i] = __builtin_amdgcn_exp2f(fmaf(s[t][i], c2, -shift));
                sum += s[t][i];
            }
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const AttnFrag<TERMS> p = half_of<TERMS>(s[t], g);
#pragma unroll
                for (int dt = 0; dt < DP / 32; ++dt)
                    attn_mma<TERMS>(acc[dt], tile_v.columns(32 * t + 16 * g, 32 * dt, lane), p);
            }
        }
    }
    sum = pccnn_add_row_xor32(sum);
    if (row >= b.rows) return;
    const int64_t token = b.query(a, row) * a.heads + b.head_of(a, row);
    if (a.splits > 1) {
        const int64_t at = (int64_t)b.split * a.m * a.heads + token;
        write_column<float, DP>(a.part + at * a.width, acc, 1.0f, half, a.width);
        if (half == 0) a.part_ml[at] = make_float2(top, sum);
    } else {
        const bool none = top == -INFINITY;                          // no live key at all: zeros
        write_column<T, DP>((T *)a.out + token * a.width, acc, none ? 0.0f : 1.0f / sum, half, a.width);
        if (a.lse != nullptr && half == 0) a.lse[token] = none ? -INFINITY : top * (1.0f / kLog2e) + logf(sum);
    }
}

// Joins the parts of a forward pass that was split over the keys: one thread per feature.
template <typename T> __global__ __launch_bounds__(kThreads) void attention_join_kernel(AttnArgs a)
{
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x, tokens = a.m * a.heads;
    if (i >= tokens * a.width) return;
    const int64_t token = i / a.width;
    float top = -INFINITY;
    for (int s = 0; s < a.splits; ++s) top = fmaxf(top, a.part_ml[s * tokens + token].x);
    const float shift = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f, value = 0.0f;
    for (int s = 0; s < a.splits; ++s) {
        const float2 ml = a.part_ml[s * tokens + token];
        const float w = __builtin_amdgcn_exp2f(ml.x - shift);
        sum = fmaf(ml.y, w, sum);
        value = fmaf(a.part[s * tokens * a.width + i], w, value);
    }
    const float one[1] = {top == -INFINITY ? 0.0f : value / sum};
    pccnn_store<1>((T *)a.out + i, one);
    if (a.lse != nullptr && i % a.width == 0)
        a.lse[token] = top == -INFINITY ? -INFINITY : top * (1.0f / kLog2e) + logf(sum);
}

// ------------------------------------------------------------------------------------------------- backward

// delta[m, heads] = dO . O, eight lanes to a row.
template <typename T>
__global__ __launch_bounds__(kThreads) void attention_delta_kernel(AttnArgs a, const T *__restrict__ out)
{
    const int64_t token = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / 8;
    const bool live = token < a.m * a.heads;
    const int64_t query = token / a.heads;
    float sum = 0.0f;
    if (live)
        for (int col = threadIdx.x % 8; col < a.width; col += 8) {
            float x[1], g[1];
            pccnn_load<1>(out + token * a.width + col, x);
            pccnn_load<1>((const T *)a.g + query * a.g_n + (token - query * a.heads) * a.g_h + col, g);
            sum = fmaf(x[0], g[0], sum);
        }
    sum = pccnn_group_sum<8>(sum);
    if (live && threadIdx.x % 8 == 0) a.delta[token] = sum;
}

template <typename T, int DP>
__global__ __launch_bounds__(kThreads) void attention_dq_kernel(AttnArgs a)
{
    constexpr int TERMS = AttnTerms<T>::value;
    extern __shared__ __align__(16) uint16_t lds[];
    const AttnTile<TERMS, kTile, DP> tile_k = {lds}, tile_v = {lds + TERMS * AttnTile<TERMS, kTile, DP>::PLANE};
    const AttnBlock b(a, blockIdx.x);
    if (b.tile * kOwn >= b.rows) return;
    const int lane = threadIdx.x % PCCNN_WAVE, wave = threadIdx.x / PCCNN_WAVE, half = lane >> 5;
    const int row = b.tile * kOwn + wave * 32 + (lane & 31);
    const bool working = b.tile * kOwn + wave * 32 < b.rows;
    const T *k = (const T *)a.k + b.k0 * a.k_n + b.head * a.k_h;
    const T *v = (const T *)a.v + b.k0 * a.v_n + b.head * a.v_h;
    const int64_t query = b.query(a, row < b.rows ? row : 0);
    const int head = b.head_of(a, row < b.rows ? row : 0);
    const int64_t token = query * a.heads + head;

    AttnFrag<TERMS> q[DP / 16], g[DP / 16];
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) {
        AttnChunk<T> c;
        attn_clear(c);
        if (row < b.rows)
            attn_load(c, (const T *)a.q + query * a.q_n + head * a.q_h, 16 * kk + 8 * half, a.width, a.wide_q);
        q[kk] = attn_frag(c);
        attn_clear(c);
        if (row < b.rows)
            attn_load(c, (const T *)a.g + query * a.g_n + head * a.g_h, 16 * kk + 8 * half, a.width, a.wide_g);
        g[kk] = attn_frag(c);
    }
    const float lse = row < b.rows ? a.lse[token] : -INFINITY, delta = row < b.rows ? a.delta[token] : 0.0f;
    const float shift = lse == -INFINITY ? INFINITY : lse * kLog2e;  // a row without keys: every P is zero
    const float c2 = a.scale * kLog2e;
    pccnn_f32x16 acc[DP / 32];
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt) clear(acc[dt]);

    int key = b.split * a.per_split * kTile;
    const int end = min(b.keys, key + a.per_split * kTile);
    Carrier<T, DP> next_k, next_v;
    uint64_t next_live = 0;
    if (key < end) {
        next_k.load(k, a.k_n, key, b.keys, a.width, a.wide_k);
        next_v.load(v, a.v_n, key, b.keys, a.width, a.wide_v);
        next_live = live_keys(a, b, key, lane);
    }
    for (; key < end; key += kTile) {
        const uint64_t live = next_live;
        __syncthreads();
        next_k.put(tile_k, live);
        next_v.put(tile_v, live);
        __syncthreads();
        if (key + kTile < end) {
            next_k.load(k, a.k_n, key + kTile, b.keys, a.width, a.wide_k);
            next_v.load(v, a.v_n, key + kTile, b.keys, a.width, a.wide_v);
            next_live = live_keys(a, b, key + kTile, lane);
        }
        if (!working || live == 0) continue;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            pccnn_f32x16 s, dp;
            clear(s);
            clear(dp);
#pragma unroll
            for (int kk = 0; kk < DP / 16; ++kk) {
                attn_mma<TERMS>(s, tile_k.rows(32 * t + (lane & 31), 16 * kk + 8 * half), q[kk]);
                attn_mma<TERMS>(dp, tile_v.rows(32 * t + (lane & 31), 16 * kk + 8 * half), g[kk]);
            }
            if (live != ~0ull) hide(s, (uint32_t)(live >> (32 * t)), half);
#pragma unroll
            for (int i = 0; i < 16; ++i)
                s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], c2, -shift)) * (dp[i] - delta);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const AttnFrag<TERMS> ds = half_of<TERMS>(s, h);
#pragma unroll
                for (int dt = 0; dt < DP / 32; ++dt)
                    attn_mma<TERMS>(acc[dt], tile_k.columns(32 * t + 16 * h, 32 * dt, lane), ds);
            }
        }
    }
    if (row >= b.rows) return;
    if (lse == -INFINITY) {                                          // whatever its gradient holds (0 times NaN)
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt) clear(acc[dt]);
    }
    if (a.splits > 1)
        write_column<float, DP>(a.part + ((int64_t)b.split * a.m * a.heads + token) * a.width, acc, a.scale, half, a.width);
    else
        write_column<T, DP>((T *)a.out + token * a.width, acc, a.scale, half, a.width);
}

template <typename T, int DP>
__global__ __launch_bounds__(kThreads) void attention_dkv_kernel(AttnArgs a)
{
    constexpr int TERMS = AttnTerms<T>::value;
    constexpr int PLANES = TERMS * AttnTile<TERMS, kTile, DP>::PLANE;
    extern __shared__ __align__(16) uint16_t lds[];
    const AttnTile<TERMS, kTile, DP> tile_q = {lds}, tile_g = {lds + PLANES};
    float *row_shift = (float *)(lds + 2 * PLANES), *row_delta = row_shift + kTile;
    const AttnBlock b(a, blockIdx.x);
    if (b.tile * kOwn >= b.keys) return;
    const int lane = threadIdx.x % PCCNN_WAVE, wave = threadIdx.x / PCCNN_WAVE, half = lane >> 5;
    const int key = b.tile * kOwn + wave * 32 + (lane & 31);
    const bool working = b.tile * kOwn + wave * 32 < b.keys;
    const bool live = key < b.keys && (a.mask == nullptr || a.mask[b.k0 + key] != 0);
    const T *q = (const T *)a.q + b.q0 * a.q_n + b.head * a.group * a.q_h;
    const T *g = (const T *)a.g + b.q0 * a.g_n + b.head * a.group * a.g_h;

    AttnFrag<TERMS> k[DP / 16], v[DP / 16];
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) {
        AttnChunk<T> c;
        attn_clear(c);
        if (live) attn_load(c, (const T *)a.k + (b.k0 + key) * a.k_n + b.head * a.k_h, 16 * kk + 8 * half, a.width, a.wide_k);
        k[kk] = attn_frag(c);
        attn_clear(c);
        if (live) attn_load(c, (const T *)a.v + (b.k0 + key) * a.v_n + b.head * a.v_h, 16 * kk + 8 * half, a.width, a.wide_v);
        v[kk] = attn_frag(c);
    }
    pccnn_f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt) {
        clear(dk[dt]);
        clear(dv[dt]);
    }
    const float c2 = a.scale * kLog2e;
    int row = (int)min((int64_t)b.split * a.per_split * kTile, (int64_t)b.rows);
    const int end = (int)min((int64_t)b.rows, row + (int64_t)a.per_split * kTile);
    Carrier<T, DP> next_q, next_g;
    float next_shift = INFINITY, next_delta = 0.0f;                  // of row threadIdx.x of the tile
    auto fetch = [&](int from) {
        next_q.load_rows(q, a.q_n, a.q_h, from, b.rows, a.group, a.width, a.wide_q);
        next_g.load_rows(g, a.g_n, a.g_h, from, b.rows, a.group, a.width, a.wide_g);
        if (threadIdx.x < kTile) {
            const int r = from + (int)threadIdx.x;
            next_shift = INFINITY;                                   // no such row, or one without keys: every P is zero
            next_delta = 0.0f;
            if (r < b.rows) {
                const int64_t token = b.query(a, r) * a.heads + b.head_of(a, r);
                const float lse = a.lse[token];
                if (lse != -INFINITY) {
                    next_shift = lse * kLog2e;
                    next_delta = a.delta[token];
                }
            }
        }
    };
    if (row < end) fetch(row);
    for (; row < end; row += kTile) {
        __syncthreads();
        next_q.put(tile_q, ~0ull);
        next_g.put(tile_g, ~0ull);
        if (threadIdx.x < kTile) {
            row_shift[threadIdx.x] = next_shift;
            row_delta[threadIdx.x] = next_delta;
        }
        __syncthreads();
        if (row + kTile < end) fetch(row + kTile);
        if (!working) continue;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            pccnn_f32x16 s, dp;
            clear(s);
            clear(dp);
#pragma unroll
            for (int kk = 0; kk < DP / 16; ++kk) {
                attn_mma<TERMS>(s, tile_q.rows(32 * t + (lane & 31), 16 * kk + 8 * half), k[kk]);
                attn_mma<TERMS>(dp, tile_g.rows(32 * t + (lane & 31), 16 * kk + 8 * half), v[kk]);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int r = 32 * t + 8 * (i / 4) + 4 * half + i % 4;
                s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], c2, -row_shift[r]));
                dp[i] = s[i] * (dp[i] - row_delta[r]);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const AttnFrag<TERMS> p = half_of<TERMS>(s, h), ds = half_of<TERMS>(dp, h);
#pragma unroll
                for (int dt = 0; dt < DP / 32; ++dt) {
                    attn_mma<TERMS>(dv[dt], tile_g.columns(32 * t + 16 * h, 32 * dt, lane), p);
                    attn_mma<TERMS>(dk[dt], tile_q.columns(32 * t + 16 * h, 32 * dt, lane), ds);
                }
            }
        }
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

// Sum of the parts of a gradient, in order.
template <typename T>
__global__ __launch_bounds__(kThreads) void attention_sum_kernel(const float *__restrict__ part, int splits, int64_t count,
                                                                T *__restrict__ out)
{
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < count; i += (int64_t)gridDim.x * kThreads) {
        float sum[1] = {0.0f};
        for (int s = 0; s < splits; ++s) sum[0] += part[s * count + i];
        pccnn_store<1>(out + i, sum);
    }
}

// ------------------------------------------------------------------------------------------------- host side

int attn_check(const char *name, const pccnn_attention *p)
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
    const int64_t strides[] = {p->q_stride_n, p->q_stride_h, p->k_stride_n, p->k_stride_h, p->v_stride_n, p->v_stride_h};
    for (int64_t s : strides)
        PCCNN_REQUIRE(s >= 0, PCCNN_ERR_INVALID, "%s: a stride of %lld elements", name, (long long)s);
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
    a.splits = 1;
    return a;
}

constexpr int64_t kWantedBlocks = 1024;      // workgroups that fill the chip (four per CU)
constexpr int kLeastTiles = 4;               // tiles below which a part is not worth its join

// Tiles of the own side, and the parts the other side is cut into so that few own tiles still fill the chip.
void attn_plan(AttnArgs &a, int64_t own, int64_t other)
{
    a.tiles = (int)std::max<int64_t>(1, pccnn_ceil_div(own, kOwn));
    const int64_t base = (int64_t)a.tiles * a.key_heads * a.clouds, tiles = std::max<int64_t>(1, pccnn_ceil_div(other, kTile));
    int64_t splits = std::max<int64_t>(1, std::min(kWantedBlocks / base, tiles / kLeastTiles));
    a.per_split = (int)pccnn_ceil_div(tiles, splits);
    a.splits = (int)pccnn_ceil_div(tiles, a.per_split);
}
void attn_plan_rows(AttnArgs &a, const pccnn_attention *p) { attn_plan(a, p->max_queries * a.group, p->max_keys); }
void attn_plan_keys(AttnArgs &a, const pccnn_attention *p) { attn_plan(a, p->max_keys, p->max_queries * a.group); }

int64_t attn_blocks(const AttnArgs &a) { return (int64_t)a.tiles * a.splits * a.key_heads * a.clouds; }

template <typename KERNEL> int attn_launch(const char *name, KERNEL kernel, const AttnArgs &a, size_t lds, hipStream_t s)
{
    const int64_t blocks = attn_blocks(a);
    PCCNN_REQUIRE(blocks <= INT32_MAX, PCCNN_ERR_UNSUPPORTED, "%s: %lld workgroups", name, (long long)blocks);
    if (lds > 65536)
        PCCNN_HIP_CHECK(hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    kernel<<<(unsigned)blocks, kThreads, lds, s>>>(a);
    PCCNN_LAUNCH_CHECK();
    return PCCNN_OK;
}

template <typename T, int DP> constexpr size_t tile_bytes() { return AttnTile<AttnTerms<T>::value, kTile, DP>::BYTES; }

// Calls f(type, padded width) for the instantiation that serves this type and head width.
template <typename F> int attn_dispatch(int type, int width, F f)
{
    auto by_width = [&](auto zero) {
        if (width <= 32) return f(zero, std::integral_constant<int, 32>());
        if (width <= 64) return f(zero, std::integral_constant<int, 64>());
        if (width <= 96) return f(zero, std::integral_constant<int, 96>());
        return f(zero, std::integral_constant<int, 128>());
    };
    return type == PCCNN_TYPE_F32 ? by_width(0.0f) : by_width((uint16_t)0);
}

size_t forward_bytes(const AttnArgs &a)
{
    if (a.splits == 1) return 0;
    const size_t tokens = (size_t)a.splits * a.m * a.heads;
    return pccnn_align(tokens * a.width * sizeof(float)) + pccnn_align(tokens * sizeof(float2));
}

} // namespace

extern "C" size_t pccnn_attention_workspace_bytes(const pccnn_attention *p, int backward)
{
    if (p == nullptr || p->heads < 1 || p->key_heads < 1 || p->clouds < 1 || p->m < 0 || p->n < 0) return 256;
    AttnArgs a = attn_args(p);
    attn_plan_rows(a, p);
    if (!backward) return std::max<size_t>(256, forward_bytes(a));
    size_t rows = a.splits > 1 ? pccnn_align((size_t)a.splits * a.m * a.heads * a.width * sizeof(float)) : 0;
    attn_plan_keys(a, p);
    size_t keys = a.splits > 1 ? 2 * pccnn_align((size_t)a.splits * a.n * a.key_heads * a.width * sizeof(float)) : 0;
    return 256 + pccnn_align((size_t)a.m * a.heads * sizeof(float)) + std::max(rows, keys);
}

extern "C" int pccnn_attention_forward(const pccnn_attention *p, void *out, float *lse_out, void *workspace,
                                       size_t workspace_bytes, void *stream)
{
    const int rc = attn_check("cross_attention", p);
    if (rc != PCCNN_OK) return rc;
    if (p->m == 0 || p->clouds == 0) return PCCNN_OK;
    PCCNN_REQUIRE(out != nullptr, PCCNN_ERR_INVALID, "cross_attention: null pointer");
    const hipStream_t s = (hipStream_t)stream;
    AttnArgs a = attn_args(p);
    a.out = out;
    a.lse = lse_out;
    attn_plan_rows(a, p);
    if (a.splits > 1) {
        PccnnArena arena(workspace, workspace_bytes);
        a.part = arena.take<float>((size_t)a.splits * a.m * a.heads * a.width);
        a.part_ml = arena.take<float2>((size_t)a.splits * a.m * a.heads);
        PCCNN_REQUIRE(arena.ok(), PCCNN_ERR_WORKSPACE, "cross_attention: workspace of %zu bytes is too small",
                      workspace_bytes);
    }
    return attn_dispatch(p->type, p->width, [&](auto zero, auto dp) -> int {
        using T = decltype(zero);
        constexpr int DP = decltype(dp)::value;
        const int rc = attn_launch("cross_attention", attention_fwd_kernel<T, DP>, a, 2 * tile_bytes<T, DP>(), s);
        if (rc != PCCNN_OK || a.splits == 1) return rc;
        attention_join_kernel<T><<<(unsigned)pccnn_ceil_div(a.m * a.heads * a.width, kThreads), kThreads, 0, s>>>(a);
        PCCNN_LAUNCH_CHECK();
        return PCCNN_OK;
    });
}

extern "C" int pccnn_attention_backward(const pccnn_attention *p, const void *out, const float *lse, const void *in_grads,
                                        int64_t grads_stride_n, int64_t grads_stride_h, void *d_queries, void *d_keys,
                                        void *d_values, void *workspace, size_t workspace_bytes, void *stream)
{
    int rc = attn_check("cross_attention_grads", p);
    if (rc != PCCNN_OK) return rc;
    PCCNN_REQUIRE(grads_stride_n >= 0 && grads_stride_h >= 0, PCCNN_ERR_INVALID, "cross_attention_grads: a negative stride");
    PCCNN_REQUIRE((d_keys != nullptr) == (d_values != nullptr), PCCNN_ERR_INVALID,
                  "cross_attention_grads: the gradients of keys and values come together");
    if (p->clouds == 0 || (d_queries == nullptr && d_keys == nullptr)) return PCCNN_OK;
    PCCNN_REQUIRE(p->m == 0 || (out && lse && in_grads), PCCNN_ERR_INVALID, "cross_attention_grads: null pointer");
    const hipStream_t s = (hipStream_t)stream;
    AttnArgs a = attn_args(p);
    a.g = in_grads;
    a.g_n = grads_stride_n;
    a.g_h = grads_stride_h;
    a.wide_g = attn_wide(a.g, a.g_n, a.g_h, p->type, a.width);
    a.lse = (float *)lse;
    PccnnArena arena(workspace, workspace_bytes);
    a.delta = arena.take<float>((size_t)p->m * p->heads);
    const size_t after = arena.used;
    return attn_dispatch(p->type, p->width, [&](auto zero, auto dp) -> int {
        using T = decltype(zero);
        constexpr int DP = decltype(dp)::value;
        int rc = PCCNN_OK;
        auto sum_parts = [&](const float *part, int64_t count, void *to) {
            const unsigned blocks = (unsigned)std::min<int64_t>(pccnn_ceil_div(count, kThreads), 8192);
            attention_sum_kernel<T><<<blocks, kThreads, 0, s>>>(part, a.splits, count, (T *)to);
        };
        if (p->m > 0) {
            PCCNN_REQUIRE(arena.ok(), PCCNN_ERR_WORKSPACE, "cross_attention_grads: workspace of %zu bytes is too small",
                          workspace_bytes);
            const int64_t threads = a.m * a.heads * 8;
            attention_delta_kernel<T><<<(unsigned)pccnn_ceil_div(threads, kThreads), kThreads, 0, s>>>(a, (const T *)out);
            PCCNN_LAUNCH_CHECK();
        }
        if (d_queries != nullptr && p->m > 0) {
            attn_plan_rows(a, p);
            a.out = d_queries;
            const int64_t count = a.m * a.heads * a.width;
            arena.used = after;
            if (a.splits > 1) {
                a.part = arena.take<float>((size_t)a.splits * count);
                PCCNN_REQUIRE(arena.ok(), PCCNN_ERR_WORKSPACE,
                              "cross_attention_grads: workspace of %zu bytes is too small", workspace_bytes);
            }
            rc = attn_launch("cross_attention_grads", attention_dq_kernel<T, DP>, a, 2 * tile_bytes<T, DP>(), s);
            if (rc != PCCNN_OK) return rc;
            if (a.splits > 1) sum_parts(a.part, count, d_queries);
            PCCNN_LAUNCH_CHECK();
        }
        if (d_keys != nullptr && p->n > 0) {
            attn_plan_keys(a, p);
            a.d_k = d_keys;
            a.d_v = d_values;
            const int64_t count = a.n * a.key_heads * a.width;
            arena.used = after;
            if (a.splits > 1) {
                a.part = arena.take<float>((size_t)a.splits * count);
                a.part_v = arena.take<float>((size_t)a.splits * count);
                PCCNN_REQUIRE(arena.ok(), PCCNN_ERR_WORKSPACE,
                              "cross_attention_grads: workspace of %zu bytes is too small", workspace_bytes);
            }
            rc = attn_launch("cross_attention_grads", attention_dkv_kernel<T, DP>, a,
                             2 * tile_bytes<T, DP>() + 2 * kTile * sizeof(float), s);
            if (rc != PCCNN_OK) return rc;
            if (a.splits > 1) {
                sum_parts(a.part, count, d_keys);
                sum_parts(a.part_v, count, d_values);
            }
            PCCNN_LAUNCH_CHECK();
        }
        return PCCNN_OK;
    });
}
