// Linear map of rows in 8 bits: out[n, o] = (sum_k codes[n, k] weights[o, k]) scale_n scale_o + bias_o.
//
// The sums are whole numbers of 32 bits, exact in any order; what is rounded is their conversion to f32 (from 2^24 on), the
// product with the scales and the result.
//
// 65536 x 1408 x 512 to bf16: 57 us, 1.66 POP/s, matrix pipe 45 % of the cycles (tiles of 256 x 256, eleven steps each, and what
// fills and empties them); 34123 x 200 x 1000 to f32: rows laid out 7 us, product 38, bound by its 136 MB of results (3.6 TB/s);
// one row of 1408 x 512: 4 us, a launch and two trips to memory.
#include "product_tiles.h"

#include <algorithm>

namespace {

// Rows that need no tiles (1408 x 512: 17, 32, 33 and 64 rows 5.2, 5.8, 6.8 and 8.6 us, in tiles 6.2).
constexpr int kFewRows = 32;
constexpr int64_t kMostWidth = 1 << 20;

struct LinearArgs {
    ProductRows x, w;
    int64_t n, outer;
    int units;
    const float *scales, *weight_scales, *bias;
    ProductGrid grid;
    size_t lds;
    void *out;
};
template <typename T, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM *WN *PCCNN_WAVE) void linear_i8_kernel(LinearArgs a)
{
    typedef ProductNT<ProductI8, BM, BN, WM, WN, false> Product;
    typedef ProductStage<T, BM, BN, Product::THREADS> Stage;
    extern __shared__ __align__(16) uint16_t lds[];
    uint32_t row_tile, col_tile;
    if (!product_tile(a.grid, blockIdx.x, row_tile, col_tile)) return;
    const int64_t row0 = (int64_t)row_tile * BM, col0 = (int64_t)col_tile * BN;
    Product p;
    float x_scale[Product::MT];
    const ProductChannels<2, BN, Product::THREADS> channels = {(float *)((char *)lds + a.lds)};
    channels.start(0, a.weight_scales, col0, a.outer);
    channels.start(1, a.bias, col0, a.outer);
#pragma unroll
    for (int m = 0; m < Product::MT; ++m) x_scale[m] = a.scales[min(row0 + p.row_of(m), a.n - 1)];
    p.run(a.x, row0, a.w, a.w, col0, a.units, lds);
    const Stage stage = {(T *)lds};
#pragma unroll
    for (int m = 0; m < Product::MT; ++m) {
#pragma unroll
        for (int n = 0; n < Product::NT; ++n)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int col = p.col_of(n) + 8 * q + 4 * p.half;
                float v[4], weight_scales[4], bias[4];
                channels.get(0, col, weight_scales);
                channels.get(1, col, bias);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float scaled = (float)p.acc[m][n][4 * q + i] * (x_scale[m] * weight_scales[i]);
                    v[i] = a.bias != nullptr ? scaled + bias[i] : scaled;
                }
                stage.put(p.row_of(m), col, v);
            }
    }
    __syncthreads();
    stage.out(DenseRow<T>{(T *)a.out, a.outer}, row0, a.n, col0, a.outer);
}

struct LinearFew {
    FewRows x, w[1];
    int64_t n, outer, inner;
    const float *scales, *weight_scales, *bias;
    void *out;
};
template <typename OUT, int RT, int WAVES> __global__ __launch_bounds__(WAVES *PCCNN_WAVE) void linear_i8_few_kernel(LinearFew a)
{
    __shared__ pccnn_u32x4 lds[WAVES - 1][RT][PCCNN_WAVE];
    const int64_t col0 = (int64_t)blockIdx.x * 16;
    FewProduct<int8_t, 1, RT, WAVES> p;
    if (!p.run(a.x, a.n, a.w, col0, a.outer, a.inner, lds)) return;
    const int lane = threadIdx.x % PCCNN_WAVE;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        const int64_t row = 16 * r + (lane & 15);
        if (row >= a.n) continue;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t o = col0 + 4 * (lane >> 4) + i;
            if (o >= a.outer) continue;
            float v[1] = {(float)p.acc[r][0][i] * (a.scales[row] * a.weight_scales[o])};
            if (a.bias != nullptr) v[0] += a.bias[o];
            pccnn_store<1>((OUT *)a.out + row * a.outer + o, v);
        }
    }
}

template <typename T, int BM, int BN, int WM, int WN> int linear_launch(LinearArgs &a, hipStream_t s)
{
    typedef ProductNT<ProductI8, BM, BN, WM, WN, false> Product;
    a.lds = std::max(Product::lds_bytes(a.units), (size_t)BM * BN * sizeof(T));
    return product_launch("linear_8bit", linear_i8_kernel<T, BM, BN, WM, WN>,
                          a.lds + ProductChannels<2, BN, Product::THREADS>::BYTES, Product::THREADS, a, pccnn_ceil_div(a.n, BM),
                          pccnn_ceil_div(a.outer, BN), s);
}
template <typename T> int linear_tiles(LinearArgs &a, hipStream_t s)
{
    if constexpr (!std::is_same<T, float>::value)
        if (product_large(a.n, a.outer, (int64_t)a.units * 16)) return linear_launch<T, 256, 256, 2, 4>(a, s);
    if (product_small(a.n, a.outer)) return linear_launch<T, 64, 64, 2, 2>(a, s);
    return a.outer <= 64 ? linear_launch<T, 128, 64, 4, 1>(a, s) : linear_launch<T, 128, 128, 2, 2>(a, s);
}
template <typename OUT> int linear_few(const LinearFew &a, hipStream_t s)
{
    constexpr int WAVES = 8;
    const unsigned blocks = (unsigned)pccnn_ceil_div(a.outer, 16);
    if (a.n <= 16)
        linear_i8_few_kernel<OUT, 1, WAVES><<<blocks, WAVES * PCCNN_WAVE, 0, s>>>(a);
    else
        linear_i8_few_kernel<OUT, 2, WAVES><<<blocks, WAVES * PCCNN_WAVE, 0, s>>>(a);
    PCCNN_LAUNCH_CHECK();
    return PCCNN_OK;
}

// How wide rows of 8-bit values can be loaded (few_load).
int linear_wide(const void *p, int64_t inner)
{
    return inner % 16 == 0 && (uintptr_t)p % 16 == 0 ? 2 : inner % 4 == 0 && (uintptr_t)p % 4 == 0 ? 1 : 0;
}
// Whether a call lays its rows (which = 0) or weights (1) out anew: rows that are not whole 16-byte units.
bool linear_staged(const void *p, int64_t n, int64_t inner) { return n > kFewRows && (inner % 16 != 0 || (uintptr_t)p % 16 != 0); }
bool linear_sizes_ok(int64_t n, int64_t inner, int64_t outer)
{
    return n >= 0 && n <= INT32_MAX && inner >= 1 && inner <= PCCNN_MAX_INNER_8BIT && outer >= 1 && outer <= kMostWidth;
}

} // namespace

extern "C" size_t pccnn_linear_8bit_workspace_bytes(const int8_t *codes, const int8_t *weights, int64_t n, int64_t inner,
                                                    int64_t outer)
{
    if (!linear_sizes_ok(n, inner, outer)) return 256;               // (the call will refuse)
    const size_t row = (size_t)pccnn_ceil_div(inner, 16) * 16;
    return 256 + (linear_staged(codes, n, inner) ? pccnn_align(n * row) : 0) +
           (linear_staged(weights, n, inner) ? pccnn_align(outer * row) : 0);
}

extern "C" int pccnn_linear_8bit(const int8_t *codes, const float *scales, const int8_t *weights, const float *weight_scales,
                                 const float *bias, int64_t n, int64_t inner, int64_t outer, void *out, int out_type,
                                 void *workspace, size_t workspace_bytes, void *stream)
{
    const char *name = "linear_8bit";
    PCCNN_REQUIRE(pccnn_type_ok(out_type), PCCNN_ERR_UNSUPPORTED, "%s: result type %d (f32 and bf16 only)", name, out_type);
    PCCNN_REQUIRE(n >= 0 && inner >= 1 && outer >= 1, PCCNN_ERR_INVALID, "%s: n=%lld, inner=%lld, outer=%lld", name, (long long)n,
                  (long long)inner, (long long)outer);
    PCCNN_REQUIRE(linear_sizes_ok(n, inner, outer), PCCNN_ERR_UNSUPPORTED,
                  "%s: %lld rows, sums over %lld products, %lld channels (2^31 - 1, %d and 2^20 at most)", name, (long long)n,
                  (long long)inner, (long long)outer, PCCNN_MAX_INNER_8BIT);
    if (n == 0) return PCCNN_OK;
    PCCNN_REQUIRE(codes && scales && weights && weight_scales && out, PCCNN_ERR_INVALID, "%s: null pointer", name);
    PCCNN_REQUIRE((uintptr_t)out % 16 == 0, PCCNN_ERR_INVALID, "%s: a result that is not 16-byte aligned", name);
    const hipStream_t s = (hipStream_t)stream;
    if (n <= kFewRows) {
        const LinearFew a = {{codes, inner, linear_wide(codes, inner)}, {{weights, inner, linear_wide(weights, inner)}}, n,
                             outer, inner, scales, weight_scales, bias, out};
        return out_type == PCCNN_TYPE_F32 ? linear_few<float>(a, s) : linear_few<uint16_t>(a, s);
    }
    const int units = (int)pccnn_ceil_div(inner, 16);
    PccnnArena arena(workspace, workspace_bytes);
    LinearArgs a = {{codes, inner, n, 0}, {weights, inner, outer, 0}, n, outer, units, scales, weight_scales, bias, {}, 0, out};
    StageArgs stage = {};
    stage.width = inner;
    stage.units = units;
    int count = 0;
    int64_t most = 0;
    for (ProductRows *r : {&a.x, &a.w}) {
        if (!linear_staged(r->p, n, inner)) continue;
        void *to = arena.take<char>((size_t)r->rows * units * 16);
        PCCNN_REQUIRE(arena.ok(), PCCNN_ERR_WORKSPACE, "%s: workspace of %zu bytes is too small", name, workspace_bytes);
        stage.s[count++] = {r->p, inner, r->rows, linear_wide(r->p, inner), to};
        most = std::max(most, r->rows * units);
        r->p = to;
        r->stride = (int64_t)units * 16;
    }
    if (count > 0) {
        product_stage_kernel<int8_t><<<dim3(product_stage_blocks(most), (unsigned)count), 256, 0, s>>>(stage);
        PCCNN_LAUNCH_CHECK();
    }
    return out_type == PCCNN_TYPE_F32 ? linear_tiles<float>(a, s) : linear_tiles<uint16_t>(a, s);
}
