// Gated linear map of feature rows, forward and backward: both projections, the activation and the product in one kernel.
//
//   G = x Wg^T   U = x Wu^T   h = act(G) U                                     x [n, c], Wg and Wu [hidden, c]
//   dG = dh U act'(G)   dU = dh act(G)   dx = dG Wg + dU Wu   dWg = dG^T x   dWu = dU^T x
//
// Nothing is kept for the backward pass but the inputs: it forms G and U anew in the kernel that turns dh into dG and dU.  Kept, they
// would be 740 MB of f32 for 65536 x 512 -> 1408, written and read again (143 us each); the products are 119 us at the rate of a large
// one.
//
// bf16 65536 x 512 -> 1408 (189 GFLOP a product), by machine: forward 205 to 245 us, dG and dU 267 to 321, dx 165 to 193, weights 178 to
// 208 and 11 for their sum: 0.59 to 1.15 PFLOP/s.  The matrix pipe works 47, 35, 62 and 63 % of the busy cycles, at 1.7 GHz: while a
// tile of 256 x 256 is filled, activated and stored nothing multiplies, since one workgroup fills a compute unit's LDS.  f32
// 32000 x 512 -> 1408, six products of terms (554 GFLOP): forward 559 to 583 us, matrix pipe 51 % at 1.9 GHz, for the same reason
// (tiles of 128 x 128 in three planes, one workgroup to a compute unit).  800000 x 64 -> 256, gelu: 150 to 171 us, vector ALU 100 %:
// 205 million results.
//
// bf16: dG and dU are rounded to bf16, since they are operands of the next products; the three gradients are then off by 0.0023 to
// 0.0025 in the 2-norm, the plain formula's by 0.0017, which is their last rounding.  Two terms of each instead would double both
// products and the 370 MB that hold them.
#include "product_tiles.h"

#include <algorithm>
#include <math.h>

namespace {

constexpr int kThreads = 256;
constexpr int64_t kMostWidth = 1 << 20;      // channels and hidden channels: a tile's rows stay within 32-bit offsets
// Rows that need no tiles: up to 32 of bf16 (512 -> 1408, 17, 32, 33 and 64 rows 5.3, 5.5, 6.9 and 7.5 us, in tiles 5.6), up to 64 of
// f32, whose operands are laid out for tiles (8.5 to 12.4 against 22).  8 bits, by how wide all three operands' rows can be loaded
// (wide_of), us without tiles : in tiles.  Whole 16 bytes: 16 and 17 rows of 512 -> 1408 3.6 : 4.2 and 4.5 : 4.2, from 1024
// channels on 32 (1024 -> 2736 17 and 32 rows 5.3 : 5.5 and 5.7 : 5.5, 1280 -> 2048 5.7 : 6.0 and 6.1 : 6.1).  Whole 4 bytes, which
// tiles lay out first: 32 (500 -> 1408 5.7 : 7.2, 1000 -> 2736 8.7 : 11.5).  Single bytes: 16 up to 512 channels (333 -> 900 6.9 : 7.5,
// 17 rows 8.8 : 7.5; one row of 501 -> 2048 7.7 : 8.6, of 701 -> 700 11.8 : 8.5, of 1365 -> 512 19 : 10).
constexpr int64_t few_rows(int type, int64_t channels, int wide)
{
    if (type != PCCNN_TYPE_I8) return type == PCCNN_TYPE_F32 ? 64 : 32;
    if (wide == 0) return channels <= 512 ? 16 : 0;
    return wide == 1 || channels >= 1024 ? 32 : 16;
}

// ------------------------------------------------------------------------------------------- activations

// Phi(x), the normal distribution function, and its density, to f32.
__device__ __forceinline__ void normal_of(float x, float &phi, float &density)
{
    density = 0.3989422804014327f * expf(-0.5f * x * x);
    phi = 0.5f * erfcf(-0.7071067811865476f * x);
}
// To what a bf16 result shows: Phi(-|x|) = (a1 t + .. + a6 t^6) exp(-x^2 / 2), t = 1 / (1 + k |x|), the form of Abramowitz and Stegun
// 7.1.26.  Their five coefficients keep the absolute error small alone (2 % of Phi(-10)); these six, and k, come from a linear program
// for the least largest error in units of 8e-8 or 2^-13 of the value, whichever is less: 2e-7 in f32 and 2^-13.5 of the value up to 13,
// where a bf16 result's own rounding is 2^-8.  `shrunk` = t exp(-x^2 / 2): one exponential, one reciprocal and some dozen other
// instructions, where a call of erfcf is some sixty and 205 million results (800000 x 256) took 250 us with it.
__device__ __forceinline__ float normal_tail(float x, float &shrunk, float &bell)
{
    const float t = __builtin_amdgcn_rcpf(fmaf(0.290968627f, fabsf(x), 1.0f));
    bell = __builtin_amdgcn_exp2f(x * x * -0.7213475204444817f);
    float p = fmaf(-0.0882386679f, t, 0.279500588f);
    p = fmaf(p, t, -0.0869634213f);
    p = fmaf(p, t, 0.176642854f);
    p = fmaf(p, t, 0.101868027f);
    p = fmaf(p, t, 0.117190566f);
    shrunk = t * bell;
    return p;
}
// act(g) and, if asked for, its derivative.  EXACT: to f32, else to what a bf16 result shows.
template <bool EXACT, bool SLOPE, int which> __device__ __forceinline__ float activate(float g, float &slope)
{
    if constexpr (which == PCCNN_ACT_RELU) {
        if (SLOPE) slope = g > 0.0f ? 1.0f : 0.0f;
        return g > 0.0f ? g : g != g ? g : 0.0f;
    }
    if constexpr (which == PCCNN_ACT_GELU) {
        if constexpr (EXACT) {
            float phi, density;
            normal_of(g, phi, density);
            if (SLOPE) slope = fmaf(g, density, phi);
            return g * phi;
        }
        float shrunk, bell;
        const float p = normal_tail(g, shrunk, bell);
        if (SLOPE) {
            const float tail = p * shrunk;
            slope = fmaf(g * 0.3989422804014327f, bell, g < 0.0f ? tail : 1.0f - tail);
        }
        // max(g, 0) - |g| Phi(-|g|); `shrunk` is zero from 64 on, but not times infinity (a NaN is in it)
        return fmaf(-__builtin_amdgcn_fmed3f(fabsf(g), 0.0f, 64.0f) * shrunk, p, __int_as_float(max(__float_as_int(g), 0)));
    }
    if constexpr (SLOPE) {                   // s and 1 - s from exp(-|g|), so that neither is what the other leaves of one
        const float e = EXACT ? expf(-fabsf(g)) : __builtin_amdgcn_exp2f(fabsf(g) * -1.4426950408889634f);
        const float r = EXACT ? 1.0f / (1.0f + e) : __builtin_amdgcn_rcpf(1.0f + e), q = e * r;
        const float s = g < 0.0f ? q : r, rest = g < 0.0f ? r : q;
        slope = which == PCCNN_ACT_SIGMOID ? r * q : s * fmaf(g, rest, 1.0f);
        return which == PCCNN_ACT_SIGMOID ? s : g * s;
    }
    const float s = EXACT ? 1.0f / (1.0f + expf(-g)) : __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(g * -1.4426950408889634f));
    return which == PCCNN_ACT_SIGMOID ? s : g * s;
}
// `call` with the activation as a constant: one branch for a tile, not one for a value.
template <typename CALL> __device__ __forceinline__ void by_activation(int which, CALL call)
{
    if (which == PCCNN_ACT_SILU)
        call(std::integral_constant<int, PCCNN_ACT_SILU>());
    else if (which == PCCNN_ACT_GELU)
        call(std::integral_constant<int, PCCNN_ACT_GELU>());
    else if (which == PCCNN_ACT_SIGMOID)
        call(std::integral_constant<int, PCCNN_ACT_SIGMOID>());
    else
        call(std::integral_constant<int, PCCNN_ACT_RELU>());
}

// ------------------------------------------------------------------------------------------- G and U

struct GatedArgs {
    ProductRows x, gate, up;                 // operands with whole units
    int64_t n, hidden;
    int units, activation;
    const float *x_scales, *gate_scales, *up_scales;                  // 8-bit operands
    ProductGrid grid;
    size_t lds;                              // bytes of the products' tiles and of the results
    void *out;                               // forward: h [n, hidden]
    const void *grads;                       // backward: dh
    int64_t grads_stride;
    int grads_wide;
    uint16_t *d_pre;                         // backward: rows (dG | dU) of 2 padded bf16 values, in pieces of 64 columns that lie one
    int64_t padded, d_plane;                 // behind the other; planes of terms in f32
};

// E: operands; T: result (forward), type of the tensors (backward).
template <class E, typename T, bool BACK, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM *WN *PCCNN_WAVE) void gated_kernel(GatedArgs a)
{
    typedef ProductNT<E, BM, BN, WM, WN, true> Product;
    constexpr int COLS = BN / 2, HALF = Product::NT / 2;
    constexpr bool EXACT = std::is_same<T, float>::value;
    typedef ProductStage<T, BM, COLS, Product::THREADS> Stage;
    extern __shared__ __align__(16) uint16_t lds[];
    uint32_t row_tile, col_tile;
    if (!product_tile(a.grid, blockIdx.x, row_tile, col_tile)) return;
    const int64_t row0 = (int64_t)row_tile * BM, col0 = (int64_t)col_tile * COLS;
    Product p;
    float x_scale[Product::MT];
    const ProductChannels<2, COLS, Product::THREADS> channels = {(float *)((char *)lds + a.lds)};
    if constexpr (std::is_same<E, ProductI8>::value) {
        channels.start(0, a.gate_scales, col0, a.hidden);
        channels.start(1, a.up_scales, col0, a.hidden);
#pragma unroll
        for (int m = 0; m < Product::MT; ++m) x_scale[m] = a.x_scales[min(row0 + p.row_of(m), a.n - 1)];
    }
    // dh is on its way during the last tile's products, in the room of the tile before it (training 65536 x 512 -> 1408
    // 827 us, asked for behind them 833)
    uint16_t *const room = p.run(a.x, row0, a.gate, a.up, col0, a.units, lds, [&](uint16_t *there) {
        if constexpr (BACK)
            if (a.grads_wide == 2) Stage{(T *)there}.bring((const T *)a.grads, a.grads_stride, row0, a.n, col0, a.hidden);
    });
    p.settle(a.x, row0, a.gate, a.up, col0, a.units);
    const Stage stage = {BACK ? (T *)room : (T *)lds}, second = {(T *)(room == lds ? lds + Product::STAGE : lds)};
    if constexpr (BACK) {
        static_assert(Stage::BYTES <= Product::STAGE * sizeof(uint16_t), "results in the tiles' rooms");
        if (a.grads_wide != 2) {
            stage.copy((const T *)a.grads, a.grads_stride, row0, a.n, col0, a.hidden);
            __syncthreads();
        }
    }
    by_activation(a.activation, [&](auto which) {
#pragma unroll
    for (int m = 0; m < Product::MT; ++m) {
        const int row = p.row_of(m);
#pragma unroll
        for (int n = 0; n < HALF; ++n)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int col = p.col_of(n) + 8 * q + 4 * p.half;
                float v[4], w[4], gate_scales[4], up_scales[4];
                if constexpr (BACK) stage.get(row, col, v);
                if constexpr (std::is_same<E, ProductI8>::value) {
                    channels.get(0, col, gate_scales);
                    channels.get(1, col, up_scales);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float g = p.acc[m][n][4 * q + i], u = p.acc[m][n + HALF][4 * q + i], slope;
                    if constexpr (std::is_same<E, ProductI8>::value) {
                        g *= x_scale[m] * gate_scales[i];
                        u *= x_scale[m] * up_scales[i];
                    }
                    const float act = activate<EXACT, BACK, decltype(which)::value>(g, slope);
                    if constexpr (BACK) {
                        w[i] = v[i] * act;
                        v[i] *= u * slope;
                    } else {
                        v[i] = act * u;
                    }
                }
                if constexpr (BACK) {                                 // channels that only fill up a unit
                    if (col0 + col + 4 > a.hidden)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (col0 + col + i >= a.hidden) v[i] = w[i] = 0.0f;
                }
                stage.put(row, col, v);
                if constexpr (BACK) second.put(row, col, w);
            }
    }
    });
    __syncthreads();
    if constexpr (!BACK) {
        stage.out(DenseRow<T>{(T *)a.out, a.hidden}, row0, a.n, col0, a.hidden);
    } else if constexpr (!EXACT) {
        stage.out(PieceRow<T>{a.d_pre, a.n, 0}, row0, a.n, col0, a.padded);
        second.out(PieceRow<T>{a.d_pre, a.n, a.padded}, row0, a.n, col0, a.padded);
    } else {
        for (int i = threadIdx.x; i < 2 * BM * COLS / 8; i += Product::THREADS) {
            const int which = i / (BM * COLS / 8), r = i % (BM * COLS / 8) / (COLS / 8), col = i % (COLS / 8) * 8;
            if (row0 + r >= a.n || col0 + col >= a.padded) continue;
            const Stage &from = which ? second : stage;
            float x[8], y[4];
            from.get(r, col, y);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = y[e];
            from.get(r, col + 4, y);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[4 + e] = y[e];
            const AttnFrag<3> f = attn_split<3, true>(x);
            uint16_t *to = PieceRow<uint16_t>{a.d_pre, a.n, which * a.padded}.at(row0 + r, col0 + col);
#pragma unroll
            for (int t = 0; t < 3; ++t) *(pccnn_u32x4 *)(to + t * a.d_plane) = __builtin_bit_cast(pccnn_u32x4, f.t[t]);
        }
    }
}

struct GatedFew {
    FewRows x, w[2];
    int64_t n, hidden, channels;
    const float *x_scales, *gate_scales, *up_scales;
    int activation;
    void *out;
};
template <typename T, typename OUT, int RT, int WAVES>
__global__ __launch_bounds__(WAVES *PCCNN_WAVE) void gated_few_kernel(GatedFew a)
{
    __shared__ pccnn_u32x4 lds[WAVES - 1][RT * 2][PCCNN_WAVE];
    const int64_t col0 = (int64_t)blockIdx.x * 16;
    FewProduct<T, 2, RT, WAVES> p;
    if (!p.run(a.x, a.n, a.w, col0, a.hidden, a.channels, lds)) return;
    const int lane = threadIdx.x % PCCNN_WAVE;
    by_activation(a.activation, [&](auto which) {
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        const int64_t row = 16 * r + (lane & 15);
        if (row >= a.n) continue;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t channel = col0 + 4 * (lane >> 4) + i;
            if (channel >= a.hidden) continue;
            float g = p.acc[r][0][i], u = p.acc[r][1][i], slope;
            if constexpr (std::is_same<T, int8_t>::value) {
                g *= a.x_scales[row] * a.gate_scales[channel];
                u *= a.x_scales[row] * a.up_scales[channel];
            }
            const float h[1] = {activate<std::is_same<OUT, float>::value, false, decltype(which)::value>(g, slope) * u};
            pccnn_store<1>((OUT *)a.out + row * a.hidden + channel, h);
        }
    }
    });
}

// ------------------------------------------------------------------------------------------- backward products

// Both weights one below the other and turned: row c of the result is (Wg[:, c] | Wu[:, c]), each padded to whole units with
// zeros.  f32: three planes of terms.  In one launch with the operands that are laid out anew (f32 training 3885 x 96 -> 256 57
// us, in two launches 62, before dx and the weights' gradients shared one).
struct TurnArgs {
    const void *gate, *up;
    int64_t gate_stride, up_stride, hidden, channels, padded;
    uint16_t *to;
    uint32_t tiles_c, blocks;                // tiles of 64 channels; workgroups that turn (both weights'), the first of the launch
    uint32_t stage_blocks;                   // and those behind them for each operand
};
template <typename T> __global__ __launch_bounds__(kThreads) void gated_prepare_kernel(TurnArgs a, StageArgs stage)
{
    __shared__ float tile[64][65];
    uint32_t block = blockIdx.x;
    if (block >= a.blocks) {
        block -= a.blocks;
        const uint32_t which = block / a.stage_blocks;
        product_stage<T>(stage, which, block - which * a.stage_blocks, a.stage_blocks);
        return;
    }
    const bool up = block >= a.blocks / 2;
    if (up) block -= a.blocks / 2;
    const int64_t c0 = (int64_t)(block % a.tiles_c) * 64, h0 = (int64_t)(block / a.tiles_c) * 64;
    const T *from = (const T *)(up ? a.up : a.gate);
    const int64_t stride = up ? a.up_stride : a.gate_stride;
#pragma unroll
    for (int j = 0; j < 64 * 64 / kThreads; ++j) {
        const int i = threadIdx.x + j * kThreads;
        const int64_t h = h0 + i / 64, c = c0 + i % 64;
        float v[1];                          // (loaded unasked, so that all loads are on their way at once)
        pccnn_load<1>(from + min(h, a.hidden - 1) * stride + min(c, a.channels - 1), v);
        tile[i / 64][i % 64] = h < a.hidden && c < a.channels ? v[0] : 0.0f;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 64 * 8; i += kThreads) {
        const int64_t c = c0 + i / 8, h = h0 + i % 8 * 8;
        if (c >= a.channels || h >= a.padded) continue;
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = tile[i % 8 * 8 + e][i / 8];
        constexpr int TERMS = AttnTerms<T>::value;
        const AttnFrag<TERMS> f = attn_split<TERMS, TERMS == 3>(x);
#pragma unroll
        for (int t = 0; t < TERMS; ++t)
            *(pccnn_u32x4 *)(a.to + (t * a.channels + c) * 2 * a.padded + (up ? a.padded : 0) + h) =
                __builtin_bit_cast(pccnn_u32x4, f.t[t]);
    }
}

template <typename T> struct ProductOf { typedef ProductBf16 type; };
template <> struct ProductOf<float> { typedef ProductF32 type; };

// dx: rows of (dG | dU) times the turned weights.  Where its tiles leave compute units without work, the sums over hidden channels
// are cut into parts that are added afterwards in their order.
struct BackArgs {
    ProductRows x, w;
    int64_t n, cols;
    int units;                               // of a part
    int all_units, splits;
    ProductGrid grid;
    void *out;                               // [n, cols], f32 [split][n, cols] of parts
};
// OUT: result, f32 for parts.
template <typename T, typename OUT, int BM, int BN, int WM, int WN>
__device__ __forceinline__ void dx_tile(const BackArgs &a, uint32_t block, uint16_t *lds)
{
    typedef ProductNT<typename ProductOf<T>::type, BM, BN, WM, WN, false> Product;
    typedef ProductStage<OUT, BM, BN, Product::THREADS> Stage;
    uint32_t row_tile, col_tile, split = 0;
    if (!product_tile(a.grid, block, row_tile, col_tile)) return;
    ProductRows x = a.x, w = a.w;
    int units = a.units;
    if (a.splits > 1) {                      // (parts are whole pieces of 128 bytes)
        split = product_split(col_tile, a.splits);
        const int first = (int)split * a.units;
        x.p = (const char *)x.p + first / 8 * x.step;
        w.p = (const char *)w.p + first / 8 * w.step;
        units = min(units, a.all_units - first);
    }
    const int64_t row0 = (int64_t)row_tile * BM, col0 = (int64_t)col_tile * BN;
    Product p;
    p.run(x, row0, w, w, col0, units, lds);
    p.settle(x, row0, w, w, col0, units);
    const Stage stage = {(OUT *)lds};
#pragma unroll
    for (int m = 0; m < Product::MT; ++m)
#pragma unroll
        for (int n = 0; n < Product::NT; ++n)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                float v[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = p.acc[m][n][4 * q + i];
                stage.put(p.row_of(m), p.col_of(n) + 8 * q + 4 * p.half, v);
            }
    __syncthreads();
    stage.out(DenseRow<OUT>{(OUT *)a.out + split * a.n * a.cols, a.cols, a.splits > 1}, row0, a.n, col0, a.cols);
}
template <typename T, typename OUT, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM *WN *PCCNN_WAVE) void gated_dx_kernel(BackArgs a)
{
    extern __shared__ __align__(16) uint16_t lds[];
    dx_tile<T, OUT, BM, BN, WM, WN>(a, blockIdx.x, lds);
}

// dWg and dWu: columns of (dG | dU) times columns of x, the inner dimension over the rows, which are cut into parts whose sums
// are added afterwards in their order.
struct WeightsArgs {
    ProductRows x, d;                        // rows with whole units; stride in bytes
    int64_t n, cols_x, cols_d;               // columns that exist, in whole units
    int tiles_x, tiles_d, splits, run;
    int64_t blocks;
    int64_t per_split;                       // rows of a part, a multiple of 64
    float *part;                             // [split][cols_d][channels]
    int64_t channels;
};

// Brings ROWS rows of up to 128 columns each into LDS, where the transposing reads take their columns; TERMS planes.
template <int ROWS, int COLS, int THREADS, int TERMS> struct ColumnsFeeder {
    typedef AttnTile<1, ROWS, COLS> Tile;
    static constexpr int ROUNDS = (ROWS * Tile::UNITS + THREADS - 1) / THREADS, COUNT = ROUNDS * TERMS;
    static constexpr int ELEMENTS = TERMS * Tile::PLANE;
    static_assert(THREADS / Tile::UNITS % 16 == 0 && (ROUNDS == 1 || ROUNDS * THREADS == ROWS * Tile::UNITS),
                  "whole wavefronts, the same unit in every round");
    const char *at;                          // the rows that are asked for next (the same in all lanes)
    int64_t step, plane;
    uint32_t off[ROUNDS];                    // the lane's units, in bytes
    int row;
    bool mine;
    // (columns of 64 a piece where the rows do not lie in one)
    __device__ __forceinline__ void start(const ProductRows &s, int64_t first, int64_t col0, int64_t cols)
    {
        row = (int)threadIdx.x / Tile::UNITS;
        const int unit = Tile::unit_at(row % ROWS, (int)threadIdx.x % Tile::UNITS);
        mine = ROWS * Tile::UNITS >= THREADS || __builtin_amdgcn_readfirstlane(threadIdx.x) < ROWS * Tile::UNITS;
        at = (const char *)s.p + first * s.stride + col0 / 64 * s.step;
        plane = s.plane;
        step = ROWS * s.stride;
#pragma unroll
        for (int j = 0; j < ROUNDS; ++j)
            off[j] = col0 + 8 * unit < cols ? (uint32_t)((row + j * (THREADS / Tile::UNITS)) * (int)s.stride + 16 * unit) : kAttnNowhere;
    }
    // The next rows; `rows`: how many of them exist.  Parts as RowsFeeder has them.
    template <int ALL> __device__ __forceinline__ void fetch(int first, int part, int rows, uint16_t *tile) const
    {
        if (!mine) return;
        const int wave_unit = __builtin_amdgcn_readfirstlane(threadIdx.x & ~(PCCNN_WAVE - 1));
#pragma unroll
        for (int t = 0; t < TERMS; ++t) {
            const __amdgpu_buffer_rsrc_t window = product_window(at + t * plane);
#pragma unroll
            for (int j = 0; j < ROUNDS; ++j)
                if ((first + t * ROUNDS + j) * 2 / ALL == part)
                    attn_bring(window, row + j * (THREADS / Tile::UNITS) < rows ? off[j] : kAttnNowhere,
                               tile + t * Tile::PLANE + 8 * (j * THREADS + wave_unit));
        }
    }
    __device__ __forceinline__ void next() { at += step; }
};
// DP x 64 columns of (dG | dU) times XP x XT columns of x; a wavefront has 32 MT x 64 of them.  64 rows a step, 32 of three planes.
constexpr int weights_threads(int dp, int xp, int xt, int mt) { return dp * 64 / (32 * mt) * (xp * xt / 64) * PCCNN_WAVE; }
constexpr int weights_rows(int terms) { return terms == 3 ? 32 : 64; }
template <class E, int DP, int XP, int XT, int MT> struct WeightsShape {
    static constexpr int COLS_D = DP * 64, COLS_X = XP * XT, WAVES_X = COLS_X / 64, WAVES_D = COLS_D / (32 * MT);
    static constexpr int THREADS = WAVES_X * WAVES_D * PCCNN_WAVE, TERMS = E::TERMS, ROWS = weights_rows(TERMS);
    static_assert(THREADS == weights_threads(DP, XP, XT, MT), "");
    static constexpr int STAGE = TERMS * ROWS * (COLS_D + COLS_X);    // uint16_t
    static constexpr size_t LDS = 2 * STAGE * sizeof(uint16_t);
};
template <class E, int DP, int XP, int XT, int MT>
__device__ __forceinline__ void weights_tile(const WeightsArgs &a, uint32_t at, uint32_t workgroups, uint16_t *lds)
{
    typedef WeightsShape<E, DP, XP, XT, MT> Shape;
    constexpr int WAVES_X = Shape::WAVES_X, STAGE = Shape::STAGE, TERMS = Shape::TERMS, ROWS = Shape::ROWS;
    typedef ColumnsFeeder<ROWS, 64, Shape::THREADS, TERMS> FeedD;
    typedef ColumnsFeeder<ROWS, XT, Shape::THREADS, TERMS> FeedX;
    typedef typename FeedD::Tile TileD;
    typedef typename FeedX::Tile TileX;
    const int lane = threadIdx.x % PCCNN_WAVE, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / PCCNN_WAVE), wx = wave % WAVES_X, wd = wave / WAVES_X;
    const int64_t block = pccnn_xcd_block(at, workgroups, a.run);
    if (block >= a.blocks) return;
    uint32_t split = __builtin_amdgcn_readfirstlane((uint32_t)block);
    const int64_t x0 = (int64_t)product_split(split, a.tiles_x) * Shape::COLS_X;
    const int64_t d0 = (int64_t)product_split(split, a.tiles_d) * Shape::COLS_D;
    const int64_t first = split * a.per_split;
    const int rows = (int)min(a.n - first, a.per_split);
    int left = rows;                         // of the tile that is asked for next
    FeedX fx[XP];
    FeedD fd[DP];
#pragma unroll
    for (int i = 0; i < XP; ++i) fx[i].start(a.x, first, x0 + i * XT, a.cols_x);
#pragma unroll
    for (int i = 0; i < DP; ++i) fd[i].start(a.d, first, d0 + i * 64, a.cols_d);
    pccnn_f32x16 acc[2][MT];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;
    const int total = (rows + ROWS - 1) / ROWS;
    constexpr int ALL = DP * FeedD::COUNT + XP * FeedX::COUNT;
    auto fetch = [&](int part, uint16_t *to) {
#pragma unroll
        for (int i = 0; i < DP; ++i) fd[i].template fetch<ALL>(i * FeedD::COUNT, part, left, to + i * FeedD::ELEMENTS);
#pragma unroll
        for (int i = 0; i < XP; ++i)
            fx[i].template fetch<ALL>(DP * FeedD::COUNT + i * FeedX::COUNT, part, left,
                                      to + DP * FeedD::ELEMENTS + i * FeedX::ELEMENTS);
        if (part == 0) return;
        left -= ROWS;
#pragma unroll
        for (int i = 0; i < DP; ++i) fd[i].next();
#pragma unroll
        for (int i = 0; i < XP; ++i) fx[i].next();
    };
    fetch(0, lds);
    fetch(1, lds);
    auto walk = [&](uint16_t *__restrict__ here, uint16_t *__restrict__ there, bool more) {
        pccnn_u32x4 fa[2][2][TERMS], fb[2][MT][TERMS];
        auto read = [&](int kk) {            // a step of products ahead of their use
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int t = 0; t < TERMS; ++t) {
                    const int col = 64 * wx + 32 * i;
                    fa[kk & 1][i][t] = __builtin_bit_cast(
                        pccnn_u32x4, TileX{here + DP * FeedD::ELEMENTS + col / XT * FeedX::ELEMENTS + t * TileX::PLANE}
                                         .columns(16 * kk, col % XT, lane).t[0]);
                }
#pragma unroll
            for (int j = 0; j < MT; ++j)
#pragma unroll
                for (int t = 0; t < TERMS; ++t) {
                    const int col = 32 * (MT * wd + j);
                    fb[kk & 1][j][t] = __builtin_bit_cast(
                        pccnn_u32x4, TileD{here + col / 64 * FeedD::ELEMENTS + t * TileD::PLANE}.columns(16 * kk, col % 64, lane).t[0]);
                }
        };
        constexpr int COUNT = ROWS / 16;
        static_assert(COUNT >= 2, "two parts of the next tile are asked for in between");
        read(0);
#pragma unroll
        for (int kk = 0; kk < COUNT; ++kk) {
            if (kk + 1 < COUNT) read(kk + 1);
            __builtin_amdgcn_sched_barrier(0x6);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int j = 0; j < MT; ++j) acc[i][j] = E::mma(fb[kk & 1][j], fa[kk & 1][i], acc[i][j]);
                if (i == 0 && kk < 2) {
                    __builtin_amdgcn_sched_barrier(0x6);
                    if (more) fetch(kk, there);
                    __builtin_amdgcn_sched_barrier(0x6);
                }
            }
            __builtin_amdgcn_sched_barrier(0x6);
        }
    };
    for (int step = 0; step < total; ++step) {
        product_landed();
        const int stage = step & 1;
        walk(lds + stage * STAGE, lds + (stage ^ 1) * STAGE, step + 1 < total);
    }
    if constexpr (TERMS == 3) {              // (as ProductNT::settle has it: one row of the part for each half of the wavefront)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < MT; ++j) {
                if (!product_unsettled(product_most<16>(acc[i][j]))) continue;
                const int64_t col_x = x0 + 64 * wx + 32 * i + (lane & 31), col_d = d0 + 32 * (MT * wd + j) + (lane & 31);
                const char *at_x = (const char *)a.x.p + first * a.x.stride + col_x / 64 * a.x.step + col_x % 64 * 2;
                const char *at_d = (const char *)a.d.p + first * a.d.stride + col_d / 64 * a.d.step + col_d % 64 * 2;
                auto value = [&](const char *at, const ProductRows &s, int row, bool there) {
                    float t[3] = {0.0f, 0.0f, 0.0f};
                    if (there && row < rows)
#pragma unroll
                        for (int e = 0; e < 3; ++e) t[e] = pccnn_bf16_value(*(const uint16_t *)(at + row * s.stride + e * s.plane));
                    return product_value(t[0], t[1], t[2]);
                };
                pccnn_f32x16 again = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll 4
                for (int row = 0; row < rows; row += 2)
                    again = __builtin_amdgcn_mfma_f32_32x32x2f32(value(at_d, a.d, row + half, col_d < a.cols_d),
                                                                 value(at_x, a.x, row + half, col_x < a.cols_x), again, 0, 0, 0);
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (!(fabsf(acc[i][j][e]) <= FLT_MAX)) acc[i][j][e] = again[e];
            }
    }
    float *part = a.part + split * a.cols_d * a.channels;
    // columns of x in the lanes: a store is of whole lines (gradients 4000 x 256 -> 704 bf16 53 us, with columns of (dG | dU) there,
    // 16 bytes of 32 rows to a store, 61)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int64_t c = x0 + 64 * wx + 32 * i + (lane & 31);
        if (c >= a.channels) continue;
#pragma unroll
        for (int j = 0; j < MT; ++j) {
            const int64_t d = d0 + 32 * (MT * wd + j) + 4 * half;
            float *to = part + d * a.channels + c;
            const int rows_d = (int)min(a.cols_d - d, (int64_t)32);
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (8 * (e / 4) + e % 4 < rows_d) to[(8 * (e / 4) + e % 4) * a.channels] = acc[i][j][e];
        }
    }
}
template <class E, int DP, int XP, int XT, int MT>
__global__ __launch_bounds__(weights_threads(DP, XP, XT, MT)) void gated_weights_kernel(WeightsArgs a)
{
    extern __shared__ __align__(16) uint16_t lds[];
    weights_tile<E, DP, XP, XT, MT>(a, blockIdx.x, gridDim.x, lds);
}
// Both, side by side: the first dx_workgroups workgroups have a tile of dx each, with four of their wavefronts.
template <typename T, class E, int DP, int XP, int XT, int MT>
__global__ __launch_bounds__(weights_threads(DP, XP, XT, MT)) void gated_both_kernel(BackArgs dx, WeightsArgs weights,
                                                                                    uint32_t dx_workgroups)
{
    extern __shared__ __align__(16) uint16_t lds[];
    if (blockIdx.x >= dx_workgroups)
        weights_tile<E, DP, XP, XT, MT>(weights, blockIdx.x - dx_workgroups, gridDim.x - dx_workgroups, lds);
    else if (threadIdx.x >= 4 * PCCNN_WAVE)
        return;
    else if (dx.splits > 1)
        dx_tile<T, float, 64, 64, 2, 2>(dx, blockIdx.x, lds);
    else
        dx_tile<T, T, 64, 64, 2, 2>(dx, blockIdx.x, lds);
}
// Sums of parts, `step` values apart, in their order: up to three results in one launch (blockIdx.y), four values or one to a thread.
struct SumTask {
    const float *part;
    int64_t step, count;
    int splits, vec;
    void *to;
};
struct SumArgs {
    SumTask t[3];
};
template <typename T, int VEC> __device__ __forceinline__ void sum_parts(const SumTask &t)
{
    const int64_t i = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * VEC;
    if (i >= t.count) return;
    const float *from = t.part + i;
    float sum[VEC] = {};
#pragma unroll 8
    for (int s = 0; s < t.splits; ++s) {
        float v[VEC];
        pccnn_load<VEC>(from + s * t.step, v);
#pragma unroll
        for (int e = 0; e < VEC; ++e) sum[e] += v[e];
    }
    pccnn_store<VEC>((T *)t.to + i, sum);
}
template <typename T> __global__ __launch_bounds__(kThreads) void gated_sum_kernel(SumArgs a)
{
    const SumTask t = blockIdx.y == 0 ? a.t[0] : blockIdx.y == 1 ? a.t[1] : a.t[2];
    if (t.vec == 4)
        sum_parts<T, 4>(t);
    else
        sum_parts<T, 1>(t);
}

// ------------------------------------------------------------------------------------------- host

int64_t unit_of(int type) { return type == PCCNN_TYPE_I8 ? 16 : 8; }
int wide_of(const void *p, int64_t stride, int64_t width, int type)
{
    const int bytes = type == PCCNN_TYPE_I8 ? 1 : pccnn_type_bytes(type);
    const bool whole = (uintptr_t)p % 16 == 0 && stride * bytes % 16 == 0;
    if (type == PCCNN_TYPE_I8)
        return whole && width % 16 == 0 ? 2 : (uintptr_t)p % 4 == 0 && stride % 4 == 0 && width % 4 == 0 ? 1 : 0;
    if (type == PCCNN_TYPE_F32) return whole && width % 4 == 0 ? 2 : 0;
    if (whole && width % 8 == 0) return 2;
    return (uintptr_t)p % 8 == 0 && stride % 4 == 0 && width % 4 == 0 ? 1 : 0;
}
// Whether rows are operands as they are.
bool as_they_are(const void *p, int64_t stride, int64_t width, int type)
{
    return type != PCCNN_TYPE_F32 && wide_of(p, stride, width, type) == 2 && stride <= kMostWidth;
}

struct GatedPlan {
    int64_t units;                           // 16-byte units of an operand row
    int planes;
    bool few;
    bool stage[3];                           // x, gate, up are laid out anew
    size_t bytes[3];
    int64_t rows[3];
    const void *p[3];
    int64_t stride[3];
    int64_t padded, pieces;                  // hidden channels in whole units; 64 columns of (dG | dU) each
    int tiles_x, tiles_d, splits;            // weights' gradients
    int64_t per_split;
    int dx_units, dx_splits;                 // dx: units of a part, parts
};
int gated_check(const char *name, const pccnn_gated *p)
{
    PCCNN_REQUIRE(p != nullptr, PCCNN_ERR_INVALID, "%s: null pointer", name);
    PCCNN_REQUIRE(pccnn_type_ok(p->type) || p->type == PCCNN_TYPE_I8, PCCNN_ERR_UNSUPPORTED,
                  "%s: element type %d (f32, bf16 and 8-bit integers only)", name, p->type);
    PCCNN_REQUIRE(p->activation >= PCCNN_ACT_SILU && p->activation <= PCCNN_ACT_RELU, PCCNN_ERR_UNSUPPORTED, "%s: activation %d",
                  name, p->activation);
    PCCNN_REQUIRE(p->n >= 0 && p->channels >= 1 && p->hidden >= 1 && p->feats_stride >= 0 && p->gate_stride >= 0 &&
                      p->up_stride >= 0,
                  PCCNN_ERR_INVALID, "%s: n=%lld, channels=%lld, hidden=%lld, row strides %lld, %lld, %lld", name,
                  (long long)p->n, (long long)p->channels, (long long)p->hidden, (long long)p->feats_stride,
                  (long long)p->gate_stride, (long long)p->up_stride);
    PCCNN_REQUIRE(p->n <= INT32_MAX && p->channels <= kMostWidth && p->hidden <= kMostWidth, PCCNN_ERR_UNSUPPORTED,
                  "%s: %lld rows of %lld channels, %lld hidden (2^31 - 1 rows, 2^20 channels at most)", name, (long long)p->n,
                  (long long)p->channels, (long long)p->hidden);
    PCCNN_REQUIRE(p->type != PCCNN_TYPE_I8 || p->channels <= PCCNN_MAX_INNER_8BIT, PCCNN_ERR_UNSUPPORTED,
                  "%s: sums over %lld 8-bit products (%d at most)", name, (long long)p->channels, PCCNN_MAX_INNER_8BIT);
    return PCCNN_OK;
}
GatedPlan gated_plan(const pccnn_gated *p, bool backward)
{
    GatedPlan plan = {};
    const int64_t unit = unit_of(p->type);
    plan.units = pccnn_ceil_div(p->channels, unit);
    plan.planes = p->type == PCCNN_TYPE_F32 ? 3 : 1;
    plan.p[0] = p->feats, plan.p[1] = p->gate, plan.p[2] = p->up;
    plan.stride[0] = p->feats_stride, plan.stride[1] = p->gate_stride, plan.stride[2] = p->up_stride;
    int wide = 2;
    for (int i = 0; i < 3; ++i) wide = std::min(wide, wide_of(plan.p[i], plan.stride[i], p->channels, p->type));
    plan.few = !backward && p->n <= few_rows(p->type, p->channels, wide);
    plan.rows[0] = p->n, plan.rows[1] = plan.rows[2] = p->hidden;
    for (int i = 0; i < 3; ++i) {
        plan.stage[i] = !plan.few && !as_they_are(plan.p[i], plan.stride[i], p->channels, p->type);
        plan.bytes[i] = plan.stage[i] ? (size_t)plan.planes * plan.rows[i] * plan.units * 16 : 0;
    }
    plan.padded = pccnn_ceil_div(p->hidden, 8) * 8;
    plan.pieces = pccnn_ceil_div(2 * plan.padded, 64);
    // parts enough to fill the chip, of at least four steps
    const bool f32 = p->type == PCCNN_TYPE_F32;
    const int rows = weights_rows(plan.planes);
    plan.tiles_x = (int)pccnn_ceil_div(p->channels, p->channels <= 64 ? 64 : f32 || p->channels <= 128 ? 128 : 256);
    plan.tiles_d = (int)pccnn_ceil_div(2 * plan.padded, f32 ? 128 : 256);
    const int64_t want = std::max<int64_t>(1, 256 / ((int64_t)plan.tiles_x * plan.tiles_d));
    const int64_t steps = std::max<int64_t>(1, pccnn_ceil_div(p->n, rows));
    const int64_t per = std::max<int64_t>(std::min<int64_t>(4, steps), pccnn_ceil_div(steps, want));
    plan.per_split = per * rows;
    plan.splits = (int)pccnn_ceil_div(steps, per);
    // dx: parts of at least 8 pieces of 128 bytes of f32 planes, 16 of bf16, that fill three quarters of the chip (gradients, in us, in
    // one part and in parts: 300 x 512 -> 1408 f32 88 and 70, bf16 42 and 40; 300 x 256 -> 704 f32 57 and 49, bf16 in parts of 8 pieces
    // 28.8 and 29.4; 1000 x 512 -> 1408, which two parts of 128 tiles would fill, f32 122 and 122, bf16 49 and 56)
    const int64_t tiles = pccnn_ceil_div(p->n, 64) * pccnn_ceil_div(p->channels, 64), pieces = plan.pieces;
    int64_t parts = 1;
    if (p->n > 0 && product_small(p->n, p->channels)) parts = std::max<int64_t>(1, std::min(192 / tiles, pieces / (f32 ? 8 : 16)));
    plan.dx_units = (int)(parts > 1 ? pccnn_ceil_div(pieces, parts) * 8 : 2 * plan.padded / 8);
    plan.dx_splits = (int)pccnn_ceil_div(2 * plan.padded / 8, plan.dx_units);
    return plan;
}
// Operands of the products: the tensors themselves, or their rows laid out anew in the workspace.  `turned` (nullable): where the
// turned weights go.
int gated_operands(const char *name, const pccnn_gated *p, const GatedPlan &plan, PccnnArena &arena, ProductRows (&r)[3],
                   uint16_t *turned, hipStream_t s)
{
    StageArgs a = {};
    a.width = p->channels;
    a.units = (int)plan.units;
    int count = 0;
    int64_t most = 0;
    const int bytes = p->type == PCCNN_TYPE_I8 ? 1 : pccnn_type_bytes(p->type);
    for (int i = 0; i < 3; ++i) {
        if (!plan.stage[i]) {
            r[i] = {plan.p[i], plan.stride[i] * bytes, plan.rows[i], 0};
            continue;
        }
        void *to = arena.take<char>(plan.bytes[i]);
        PCCNN_REQUIRE(arena.ok(), PCCNN_ERR_WORKSPACE, "%s: workspace of %zu bytes is too small", name, arena.size);
        r[i] = {to, plan.units * 16, plan.rows[i], plan.rows[i] * plan.units * 16};
        a.s[count++] = {plan.p[i], plan.stride[i], plan.rows[i], wide_of(plan.p[i], plan.stride[i], p->channels, p->type), to};
        most = std::max(most, plan.rows[i] * plan.units);
    }
    if (turned != nullptr) {
        TurnArgs t = {p->gate, p->up, p->gate_stride, p->up_stride, p->hidden, p->channels, plan.padded, turned};
        t.tiles_c = (uint32_t)pccnn_ceil_div(p->channels, 64);
        t.blocks = 2 * t.tiles_c * (uint32_t)pccnn_ceil_div(plan.padded, 64);
        t.stage_blocks = product_stage_blocks(most);
        const unsigned blocks = t.blocks + t.stage_blocks * count;
        if (p->type == PCCNN_TYPE_F32)
            gated_prepare_kernel<float><<<blocks, kThreads, 0, s>>>(t, a);
        else
            gated_prepare_kernel<uint16_t><<<blocks, kThreads, 0, s>>>(t, a);
    } else if (count > 0) {
        const dim3 grid(product_stage_blocks(most), (unsigned)count);
        if (p->type == PCCNN_TYPE_F32)
            product_stage_kernel<float><<<grid, 256, 0, s>>>(a);
        else if (p->type == PCCNN_TYPE_BF16)
            product_stage_kernel<uint16_t><<<grid, 256, 0, s>>>(a);
        else
            product_stage_kernel<int8_t><<<grid, 256, 0, s>>>(a);
    }
    PCCNN_LAUNCH_CHECK();
    return PCCNN_OK;
}
template <class E, typename T, bool BACK, int BM, int BN, int WM, int WN>
int gated_launch_tile(const char *name, GatedArgs &a, hipStream_t s)
{
    typedef ProductNT<E, BM, BN, WM, WN, true> Product;
    a.lds = std::max(Product::lds_bytes(a.units), BACK ? 2 * Product::STAGE * sizeof(uint16_t) : (size_t)BM * BN / 2 * sizeof(T));
    const size_t channels = std::is_same<E, ProductI8>::value ? ProductChannels<2, BN / 2, Product::THREADS>::BYTES : 0;
    return product_launch(name, gated_kernel<E, T, BACK, BM, BN, WM, WN>, a.lds + channels, Product::THREADS, a, pccnn_ceil_div(a.n, BM),
                          pccnn_ceil_div(a.hidden, BN / 2), s);
}
template <class E, typename T, bool BACK> int gated_launch(const char *name, GatedArgs &a, hipStream_t s)
{
    if (product_small(a.n, 2 * a.hidden)) return gated_launch_tile<E, T, BACK, 64, 64, 2, 1>(name, a, s);
    if constexpr (std::is_same<E, ProductF32>::value) {
        return gated_launch_tile<E, T, BACK, 128, 128, 4, 2>(name, a, s);
    } else {
        if (product_large(a.n, 2 * a.hidden, (int64_t)a.units * E::UNIT))
            return gated_launch_tile<E, T, BACK, 256, 256, 4, 2>(name, a, s);
        return gated_launch_tile<E, T, BACK, 128, 128, 2, 2>(name, a, s);
    }
}
template <typename T, int BM, int BN, int WM, int WN, typename OUT = T> int dx_launch(const char *name, BackArgs &a, hipStream_t s)
{
    typedef ProductNT<typename ProductOf<T>::type, BM, BN, WM, WN, false> Product;
    const size_t lds = std::max(Product::lds_bytes(a.units), (size_t)BM * BN * sizeof(OUT));
    return product_launch(name, gated_dx_kernel<T, OUT, BM, BN, WM, WN>, lds, Product::THREADS, a, pccnn_ceil_div(a.n, BM),
                          pccnn_ceil_div(a.cols, BN) * a.splits, s);
}
template <typename T> int dx_launch(const char *name, BackArgs &a, hipStream_t s)
{
    if (a.splits > 1) return dx_launch<T, 64, 64, 2, 2, float>(name, a, s);
    if (product_small(a.n, a.cols)) return dx_launch<T, 64, 64, 2, 2>(name, a, s);
    if constexpr (std::is_same<T, float>::value) {
        return a.cols <= 64 ? dx_launch<T, 128, 64, 4, 2>(name, a, s) : dx_launch<T, 128, 128, 4, 2>(name, a, s);
    } else {
        if (product_large(a.n, a.cols, (int64_t)a.units * 8)) return dx_launch<T, 256, 256, 4, 2>(name, a, s);
        return a.cols <= 64 ? dx_launch<T, 128, 64, 4, 1>(name, a, s) : dx_launch<T, 128, 128, 2, 2>(name, a, s);
    }
}

// A part's tiles go to one XCD as far as they may: they read the same rows, and its L2 serves them once.  `dx` (nullable): its tiles
// of 64 x 64 in the same launch.
template <typename T, class E, int DP, int XP, int XT, int MT> int weights_launch(WeightsArgs &a, BackArgs *dx, hipStream_t s)
{
    typedef WeightsShape<E, DP, XP, XT, MT> Shape;
    typedef ProductNT<E, 64, 64, 2, 2, false> Product;
    a.blocks = (int64_t)a.tiles_x * a.tiles_d * a.splits;
    a.run = (int)pccnn_ceil_div(a.blocks, PCCNN_XCDS);
    const unsigned workgroups = pccnn_xcd_grid(a.blocks, a.run);
    const void *kernel = dx != nullptr ? (const void *)gated_both_kernel<T, E, DP, XP, XT, MT>
                                       : (const void *)gated_weights_kernel<E, DP, XP, XT, MT>;
    const size_t lds = std::max(Shape::LDS, dx != nullptr ? std::max(Product::lds_bytes(dx->units), 64 * 64 * sizeof(float)) : 0);
    if (lds > 65536) PCCNN_HIP_CHECK(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    if (dx != nullptr) {
        dx->grid = product_grid(pccnn_ceil_div(dx->n, 64), pccnn_ceil_div(dx->cols, 64) * dx->splits);
        const unsigned first = product_workgroups(dx->grid);
        gated_both_kernel<T, E, DP, XP, XT, MT><<<first + workgroups, Shape::THREADS, lds, s>>>(*dx, a, first);
    } else {
        gated_weights_kernel<E, DP, XP, XT, MT><<<workgroups, Shape::THREADS, lds, s>>>(a);
    }
    PCCNN_LAUNCH_CHECK();
    return PCCNN_OK;
}

template <typename T, typename OUT> int few_launch(GatedFew &a, hipStream_t s)
{
    constexpr int WAVES = 8;
    const unsigned blocks = (unsigned)pccnn_ceil_div(a.hidden, 16);
    if (a.n <= 16)
        gated_few_kernel<T, OUT, 1, WAVES><<<blocks, WAVES * PCCNN_WAVE, 0, s>>>(a);
    else if (a.n <= 32)
        gated_few_kernel<T, OUT, 2, WAVES><<<blocks, WAVES * PCCNN_WAVE, 0, s>>>(a);
    else if constexpr (std::is_same<T, float>::value)
        gated_few_kernel<T, OUT, 4, WAVES><<<blocks, WAVES * PCCNN_WAVE, 0, s>>>(a);
    PCCNN_LAUNCH_CHECK();
    return PCCNN_OK;
}

struct BackBytes {
    size_t d_pre, turned, part, dx_part;
    size_t all() const { return pccnn_align(d_pre) + pccnn_align(turned) + pccnn_align(part) + pccnn_align(dx_part); }
};
BackBytes back_bytes(const pccnn_gated *p, const GatedPlan &plan)
{
    BackBytes b;
    b.d_pre = (size_t)plan.planes * p->n * plan.pieces * 128;
    b.turned = (size_t)plan.planes * p->channels * 2 * plan.padded * 2;
    b.part = (size_t)plan.splits * 2 * plan.padded * p->channels * sizeof(float);
    b.dx_part = plan.dx_splits > 1 ? (size_t)plan.dx_splits * p->n * p->channels * sizeof(float) : 0;
    return b;
}

} // namespace

extern "C" size_t pccnn_gated_workspace_bytes(const pccnn_gated *p, int backward)
{
    if (gated_check("gated_workspace_bytes", p) != PCCNN_OK) return 256;
    const GatedPlan plan = gated_plan(p, backward != 0);
    size_t total = 256;
    for (size_t bytes : plan.bytes) total += pccnn_align(bytes);
    if (backward && p->type != PCCNN_TYPE_I8) total += back_bytes(p, plan).all();
    return total;
}

extern "C" int pccnn_gated_forward(const pccnn_gated *p, void *out, int out_type, void *workspace, size_t workspace_bytes,
                                   void *stream)
{
    const char *name = "gated_linear";
    int rc = gated_check(name, p);
    if (rc != PCCNN_OK) return rc;
    PCCNN_REQUIRE(pccnn_type_ok(out_type) && (p->type == PCCNN_TYPE_I8 || out_type == p->type), PCCNN_ERR_UNSUPPORTED,
                  "%s: result type %d of operands of type %d", name, out_type, p->type);
    if (p->n == 0) return PCCNN_OK;
    PCCNN_REQUIRE(p->feats && p->gate && p->up && out, PCCNN_ERR_INVALID, "%s: null pointer", name);
    PCCNN_REQUIRE(p->type != PCCNN_TYPE_I8 || (p->feats_scales && p->gate_scales && p->up_scales), PCCNN_ERR_INVALID,
                  "%s: 8-bit operands without their scales", name);
    PCCNN_REQUIRE((uintptr_t)out % 16 == 0, PCCNN_ERR_INVALID, "%s: a result that is not 16-byte aligned", name);
    const hipStream_t s = (hipStream_t)stream;
    const GatedPlan plan = gated_plan(p, false);
    if (plan.few) {
        GatedFew a = {{p->feats, p->feats_stride, wide_of(p->feats, p->feats_stride, p->channels, p->type)},
                      {{p->gate, p->gate_stride, wide_of(p->gate, p->gate_stride, p->channels, p->type)},
                       {p->up, p->up_stride, wide_of(p->up, p->up_stride, p->channels, p->type)}},
                      p->n, p->hidden, p->channels, p->feats_scales, p->gate_scales, p->up_scales, p->activation, out};
        if (p->type == PCCNN_TYPE_F32) return few_launch<float, float>(a, s);
        if (p->type == PCCNN_TYPE_BF16) return few_launch<uint16_t, uint16_t>(a, s);
        return out_type == PCCNN_TYPE_F32 ? few_launch<int8_t, float>(a, s) : few_launch<int8_t, uint16_t>(a, s);
    }
    PccnnArena arena(workspace, workspace_bytes);
    ProductRows r[3];
    rc = gated_operands(name, p, plan, arena, r, nullptr, s);
    if (rc != PCCNN_OK) return rc;
    GatedArgs a = {};
    a.x = r[0], a.gate = r[1], a.up = r[2];
    a.n = p->n, a.hidden = p->hidden, a.units = (int)plan.units, a.activation = p->activation;
    a.x_scales = p->feats_scales, a.gate_scales = p->gate_scales, a.up_scales = p->up_scales;
    a.out = out;
    if (p->type == PCCNN_TYPE_F32) return gated_launch<ProductF32, float, false>(name, a, s);
    if (p->type == PCCNN_TYPE_BF16) return gated_launch<ProductBf16, uint16_t, false>(name, a, s);
    return out_type == PCCNN_TYPE_F32 ? gated_launch<ProductI8, float, false>(name, a, s)
                                      : gated_launch<ProductI8, uint16_t, false>(name, a, s);
}

extern "C" int pccnn_gated_backward(const pccnn_gated *p, const void *in_grads, int64_t grads_stride, void *d_feats, void *d_gate,
                                    void *d_up, void *workspace, size_t workspace_bytes, void *stream)
{
    const char *name = "gated_linear_grads";
    int rc = gated_check(name, p);
    if (rc != PCCNN_OK) return rc;
    PCCNN_REQUIRE(p->type != PCCNN_TYPE_I8, PCCNN_ERR_UNSUPPORTED, "%s: 8-bit operands have no gradients", name);
    PCCNN_REQUIRE(grads_stride >= 0, PCCNN_ERR_INVALID, "%s: gradient rows %lld apart", name, (long long)grads_stride);
    PCCNN_REQUIRE(p->hidden * p->channels <= INT32_MAX, PCCNN_ERR_UNSUPPORTED, "%s: weights of %lld x %lld (2^31 - 1 values at most)",
                  name, (long long)p->hidden, (long long)p->channels);
    PCCNN_REQUIRE((d_gate != nullptr) == (d_up != nullptr), PCCNN_ERR_INVALID, "%s: the gradients of both weights come together",
                  name);
    if (d_gate == nullptr && (d_feats == nullptr || p->n == 0)) return PCCNN_OK;
    PCCNN_REQUIRE(p->gate && p->up && (p->n == 0 || (p->feats && in_grads)), PCCNN_ERR_INVALID, "%s: null pointer", name);
    PCCNN_REQUIRE(((uintptr_t)d_feats | (uintptr_t)d_gate | (uintptr_t)d_up) % 16 == 0, PCCNN_ERR_INVALID,
                  "%s: a result that is not 16-byte aligned", name);
    const hipStream_t s = (hipStream_t)stream;
    const GatedPlan plan = gated_plan(p, true);
    const BackBytes bytes = back_bytes(p, plan);
    PccnnArena arena(workspace, workspace_bytes);
    ProductRows r[3];
    const bool f32 = p->type == PCCNN_TYPE_F32;
    const ProductRows d = {arena.take<char>(bytes.d_pre), 128, p->n, p->n * plan.pieces * 128, p->n * 128};
    uint16_t *turned = arena.take<uint16_t>(bytes.turned / 2);
    float *part = arena.take<float>(bytes.part / sizeof(float)), *dx_part = arena.take<float>(bytes.dx_part / sizeof(float));
    PCCNN_REQUIRE(arena.ok(), PCCNN_ERR_WORKSPACE, "%s: workspace of %zu bytes is too small", name, workspace_bytes);
    if (p->n > 0) {
        rc = gated_operands(name, p, plan, arena, r, d_feats != nullptr ? turned : nullptr, s);
        if (rc != PCCNN_OK) return rc;
        GatedArgs a = {};
        a.x = r[0], a.gate = r[1], a.up = r[2];
        a.n = p->n, a.hidden = p->hidden, a.units = (int)plan.units, a.activation = p->activation;
        a.grads = in_grads, a.grads_stride = grads_stride;
        a.grads_wide = grads_stride <= kMostWidth ? wide_of(in_grads, grads_stride, p->hidden, p->type) : 0;
        a.d_pre = (uint16_t *)d.p, a.padded = plan.padded, a.d_plane = d.plane / 2;
        rc = f32 ? gated_launch<ProductF32, float, true>(name, a, s) : gated_launch<ProductBf16, uint16_t, true>(name, a, s);
        if (rc != PCCNN_OK) return rc;
    }
    SumArgs sums = {};
    int tasks = 0;
    auto add = [&](const float *from, int64_t step, int64_t count, int splits, bool wide, void *to) {
        sums.t[tasks++] = {from, step, count, splits, wide ? 4 : 1, to};
    };
    BackArgs dx = {};
    const bool want_dx = d_feats != nullptr && p->n > 0;
    if (want_dx) {
        dx.x = d;
        dx.w = {turned, 4 * plan.padded, p->channels, p->channels * 4 * plan.padded};
        dx.n = p->n, dx.cols = p->channels, dx.out = plan.dx_splits > 1 ? (void *)dx_part : d_feats;
        dx.units = plan.dx_units, dx.all_units = (int)(2 * plan.padded / 8), dx.splits = plan.dx_splits;
        const int64_t count = p->n * p->channels;
        if (plan.dx_splits > 1) add(dx_part, count, count, plan.dx_splits, count % 4 == 0, d_feats);
    }
    // tiles of dx that leave compute units idle go with the weights' gradients: training 3885 x 96 -> 256 f32 43.7 us, one behind the
    // other 54.3, bf16 26.5 and 30.7; 4000 x 256 -> 704, where both fill the chip, bf16 51 and 52
    const bool together = want_dx && d_gate != nullptr && product_small(p->n, p->channels);
    if (want_dx && !together) {
        rc = f32 ? dx_launch<float>(name, dx, s) : dx_launch<uint16_t>(name, dx, s);
        if (rc != PCCNN_OK) return rc;
    }
    if (d_gate != nullptr) {
        if (p->n > 0) {
            WeightsArgs a = {};
            a.x = r[0], a.d = d, a.n = p->n, a.cols_x = plan.units * 8, a.cols_d = 2 * plan.padded;
            a.tiles_x = plan.tiles_x, a.tiles_d = plan.tiles_d, a.splits = plan.splits, a.per_split = plan.per_split;
            a.part = part, a.channels = p->channels;
            BackArgs *const beside = together ? &dx : nullptr;
            if (f32)
                rc = p->channels <= 64 ? weights_launch<float, ProductF32, 2, 1, 64, 1>(a, beside, s)
                                       : weights_launch<float, ProductF32, 2, 1, 128, 1>(a, beside, s);
            else
                rc = p->channels <= 64    ? weights_launch<uint16_t, ProductBf16, 4, 1, 64, 2>(a, beside, s)
                     : p->channels <= 128 ? weights_launch<uint16_t, ProductBf16, 4, 1, 128, 2>(a, beside, s)
                                          : weights_launch<uint16_t, ProductBf16, 4, 2, 128, 4>(a, beside, s);
            if (rc != PCCNN_OK) return rc;
        }
        const int64_t one = plan.padded * p->channels;
        for (int i = 0; i < 2; ++i)
            add(part + i * one, 2 * one, p->hidden * p->channels, p->n > 0 ? plan.splits : 0, p->channels % 4 == 0, i ? d_up : d_gate);
    }
    if (tasks > 0) {
        int64_t most = 0;
        for (int i = 0; i < tasks; ++i) most = std::max(most, pccnn_ceil_div(sums.t[i].count, kThreads * sums.t[i].vec));
        const dim3 grid((unsigned)most, (unsigned)tasks);
        if (f32)
            gated_sum_kernel<float><<<grid, kThreads, 0, s>>>(sums);
        else
            gated_sum_kernel<uint16_t><<<grid, kThreads, 0, s>>>(sums);
        PCCNN_LAUNCH_CHECK();
    }
    return PCCNN_OK;
}
