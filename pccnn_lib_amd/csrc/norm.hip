// Layer norm of feature rows, forward and backward.
//
//   mean = avg(x)   rstd = 1 / sqrt(avg((x - mean)^2) + eps)   xhat = (x - mean) rstd   y = xhat gamma + beta
//   s = dy gamma    dx = rstd (s - avg(s) - xhat avg(s xhat))   dgamma = sum_rows dy xhat   dbeta = sum_rows dy
//
// A row lives in the registers of LANES lanes (LANES <= 64, a wavefront works on 64 / LANES rows at a time), so the
// squares are taken of centred values and a row is read once.  A lane keeps the same columns for every row it works on:
// gamma, beta and the two column sums of the backward pass stay in registers over the whole loop, and one small second
// kernel adds the workgroups' sums in a fixed order (no atomics: the same bits from run to run).  Rows longer than a
// wavefront's registers hold (2048 values, or 1024 where rows only allow loads of single values: f32 rows that are not 16-byte
// aligned, odd channel counts) take a workgroup each and are read again from the caches instead.
//
// Bound by HBM.  800000 rows of 64 bf16 values: forward 39 us = 5.3 TB/s, backward 64 us = 4.8 TB/s (three streams, the
// column sums in registers cost nothing), sums 4 us; a copy of that size runs at 5.1 TB/s.  65536 rows of 128 f32: 13, 17 - 18
// and 3.7 us (both passes fit the 256 MB cache).  One row: 2 us, the launch.  Two rows at a time in the backward pass and
// half as many rows of sums took the last kernel from 6.6 to 3.9 us and left the first one as it was.  Single-value loads:
// 32768 rows of 1021 f32 as fast as aligned rows of 1024 (6.2 TB/s forward, 4.8 backward), of bf16 1.9 TB/s and 3.3 where aligned
// rows have 4.0 and 4.9.  A workgroup per row: 16384 rows of 2056 f32 3.5 TB/s and 2.2, of bf16 1.8 and 1.7.
#include "elements.h"

#include <algorithm>

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / PCCNN_WAVE;
constexpr int kMaxBlocks = 1024;             // workgroups of the persistent kernels: four per CU, sixteen wavefronts
// The backward pass has as many wavefronts in half as many workgroups: every one leaves a row of column sums.
constexpr int kBackThreads = 512, kBackWaves = kBackThreads / PCCNN_WAVE, kBackBlocks = 512;
constexpr int kRegisterColumns = 2048;       // the longest row that one wavefront holds (32 values per lane)
constexpr int kMostLoads = 16;               // in at most so many loads per lane: single values reach 1024

// ------------------------------------------------------------------------------------ rows in registers

template <typename T, int VEC, int LANES, int CHUNKS>
__global__ __launch_bounds__(kThreads) void norm_fwd_kernel(const T *__restrict__ feats, int64_t stride,
                                                           const void *__restrict__ gamma,
                                                           const void *__restrict__ beta, int weight_type, float eps,
                                                           int64_t n, int c, T *__restrict__ out,
                                                           float2 *__restrict__ stats)
{
    constexpr int ROWS = PCCNN_WAVE / LANES;
    const int lane = threadIdx.x % LANES, slot = (threadIdx.x % PCCNN_WAVE) / LANES;
    const int64_t first = ((int64_t)blockIdx.x * kWaves + threadIdx.x / PCCNN_WAVE) * ROWS + slot;
    const int64_t step = (int64_t)gridDim.x * kWaves * ROWS;
    const float inv_c = 1.0f / (float)c;
    float g[CHUNKS][VEC], b[CHUNKS][VEC];
#pragma unroll
    for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const int col = (k * LANES + lane) * VEC + i;
            g[k][i] = col < c ? pccnn_element(gamma, weight_type, col) : 0.0f;
            b[k][i] = col < c ? pccnn_element(beta, weight_type, col) : 0.0f;
        }
    // every lane of a wavefront runs the same number of rounds: the row sums need all of them
    for (int64_t base = first - slot; base < n; base += step) {
        const int64_t row = base + slot;
        const bool live = row < n;
        float x[CHUNKS][VEC], sum = 0.0f;
#pragma unroll
        for (int k = 0; k < CHUNKS; ++k) {
            const int col = (k * LANES + lane) * VEC;
            if (live && col < c) {
                pccnn_load<VEC>(feats + row * stride + col, x[k]);
            } else {
#pragma unroll
                for (int i = 0; i < VEC; ++i) x[k][i] = 0.0f;
            }
#pragma unroll
            for (int i = 0; i < VEC; ++i) sum += x[k][i];
        }
        const float mean = pccnn_group_sum<LANES>(sum) * inv_c;
        float squares = 0.0f;
#pragma unroll
        for (int k = 0; k < CHUNKS; ++k) {
            const bool in = (k * LANES + lane) * VEC < c;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                x[k][i] -= mean;
                if (in) squares = fmaf(x[k][i], x[k][i], squares);
            }
        }
        const float rstd = 1.0f / sqrtf(pccnn_group_sum<LANES>(squares) * inv_c + eps);
        if (!live) continue;
#pragma unroll
        for (int k = 0; k < CHUNKS; ++k) {
            const int col = (k * LANES + lane) * VEC;
            if (col < c) {
                float y[VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) y[i] = fmaf(x[k][i] * rstd, g[k][i], b[k][i]);
                pccnn_store<VEC>(out + row * c + col, y);
            }
        }
        if (stats != nullptr && lane == 0) stats[row] = make_float2(mean, rstd);
    }
}

// sums_gamma, sums_beta: a workgroup's column sums, sums_stride values after the last workgroup's, or null when nobody wants
// them; d_feats null likewise.  Short rows are worked on two at a time, so that a lane has four loads on their way.
template <typename T, int VEC, int LANES, int CHUNKS>
__global__ __launch_bounds__(kBackThreads) void norm_bwd_kernel(const T *__restrict__ feats, int64_t stride,
                                                               const void *__restrict__ gamma, int weight_type,
                                                               const float2 *__restrict__ stats,
                                                               const T *__restrict__ grads, int64_t grads_stride,
                                                               int64_t n, int c, T *__restrict__ d_feats,
                                                               float *__restrict__ sums_gamma,
                                                               float *__restrict__ sums_beta, int64_t sums_stride)
{
    constexpr int ROWS = PCCNN_WAVE / LANES;
    constexpr int COLUMNS = LANES * CHUNKS * VEC;
    constexpr int PAIR = CHUNKS * VEC <= 8 ? 2 : 1;
    __shared__ float sums[kBackWaves][COLUMNS];
    const int lane = threadIdx.x % LANES, slot = (threadIdx.x % PCCNN_WAVE) / LANES, wave = threadIdx.x / PCCNN_WAVE;
    const int64_t first = ((int64_t)blockIdx.x * kBackWaves + wave) * ROWS;
    const int64_t step = (int64_t)gridDim.x * kBackWaves * ROWS;
    const float inv_c = 1.0f / (float)c;
    float w[CHUNKS][VEC], dg[CHUNKS][VEC], db[CHUNKS][VEC];
#pragma unroll
    for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const int col = (k * LANES + lane) * VEC + i;
            w[k][i] = col < c ? pccnn_element(gamma, weight_type, col) : 0.0f;
            dg[k][i] = db[k][i] = 0.0f;
        }
    for (int64_t base = first; base < n; base += PAIR * step) {
        float x[PAIR][CHUNKS][VEC], g[PAIR][CHUNKS][VEC];
        float2 stat[PAIR];
#pragma unroll
        for (int u = 0; u < PAIR; ++u) {
            const int64_t row = base + u * step + slot;
            const bool live = row < n;
            stat[u] = live ? stats[row] : make_float2(0.0f, 0.0f);
#pragma unroll
            for (int k = 0; k < CHUNKS; ++k) {
                const int col = (k * LANES + lane) * VEC;
                if (live && col < c) {
                    pccnn_load<VEC>(feats + row * stride + col, x[u][k]);
                    pccnn_load<VEC>(grads + row * grads_stride + col, g[u][k]);
                } else {
#pragma unroll
                    for (int i = 0; i < VEC; ++i) { x[u][k][i] = stat[u].x; g[u][k][i] = 0.0f; }
                }
            }
        }
#pragma unroll
        for (int u = 0; u < PAIR; ++u) {
            const int64_t row = base + u * step + slot;
            float sum = 0.0f, dot = 0.0f;
#pragma unroll
            for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    x[u][k][i] = (x[u][k][i] - stat[u].x) * stat[u].y;
                    dg[k][i] = fmaf(g[u][k][i], x[u][k][i], dg[k][i]);
                    db[k][i] += g[u][k][i];
                    g[u][k][i] *= w[k][i];
                    sum += g[u][k][i];
                    dot = fmaf(g[u][k][i], x[u][k][i], dot);
                }
            if (d_feats == nullptr) continue;
            sum = pccnn_group_sum<LANES>(sum) * inv_c;
            dot = pccnn_group_sum<LANES>(dot) * inv_c;
            if (row >= n) continue;
#pragma unroll
            for (int k = 0; k < CHUNKS; ++k) {
                const int col = (k * LANES + lane) * VEC;
                if (col < c) {
                    float d[VEC];
#pragma unroll
                    for (int i = 0; i < VEC; ++i) d[i] = stat[u].y * (g[u][k][i] - sum - x[u][k][i] * dot);
                    pccnn_store<VEC>(d_feats + row * c + col, d);
                }
            }
        }
    }
    if (sums_gamma == nullptr) return;
    const int64_t mine = (int64_t)blockIdx.x * sums_stride;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        __syncthreads();
#pragma unroll
        for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float total = pccnn_strided_sum<LANES>(which == 0 ? dg[k][i] : db[k][i]);
                if (slot == 0) sums[wave][(k * LANES + lane) * VEC + i] = total;
            }
        __syncthreads();
        for (int col = threadIdx.x; col < c; col += kBackThreads) {
            float total = 0.0f;
#pragma unroll
            for (int v = 0; v < kBackWaves; ++v) total += sums[v][col];
            (which == 0 ? sums_gamma : sums_beta)[mine + col] = total;
        }
    }
}

// ---------------------------------------------------------------------------------------- rows of any length

__device__ __forceinline__ float block_sum(float v, float *scratch)
{
    v = pccnn_group_sum<PCCNN_WAVE>(v);
    __syncthreads();
    if (threadIdx.x % PCCNN_WAVE == 0) scratch[threadIdx.x / PCCNN_WAVE] = v;
    __syncthreads();
    float total = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) total += scratch[w];
    return total;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void norm_fwd_wide_kernel(const T *__restrict__ feats, int64_t stride,
                                                                const void *__restrict__ gamma,
                                                                const void *__restrict__ beta, int weight_type,
                                                                float eps, int64_t n, int64_t c, T *__restrict__ out,
                                                                float2 *__restrict__ stats)
{
    __shared__ float scratch[kWaves];
    for (int64_t row = blockIdx.x; row < n; row += gridDim.x) {
        const T *x = feats + row * stride;
        float v[1], sum = 0.0f, squares = 0.0f;
        for (int64_t col = threadIdx.x; col < c; col += kThreads) {
            pccnn_load<1>(x + col, v);
            sum += v[0];
        }
        const float mean = block_sum(sum, scratch) / (float)c;
        for (int64_t col = threadIdx.x; col < c; col += kThreads) {
            pccnn_load<1>(x + col, v);
            squares = fmaf(v[0] - mean, v[0] - mean, squares);
        }
        const float rstd = 1.0f / sqrtf(block_sum(squares, scratch) / (float)c + eps);
        for (int64_t col = threadIdx.x; col < c; col += kThreads) {
            pccnn_load<1>(x + col, v);
            v[0] = fmaf((v[0] - mean) * rstd, pccnn_element(gamma, weight_type, col),
                        pccnn_element(beta, weight_type, col));
            pccnn_store<1>(out + row * c + col, v);
        }
        if (stats != nullptr && threadIdx.x == 0) stats[row] = make_float2(mean, rstd);
    }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void norm_bwd_wide_kernel(const T *__restrict__ feats, int64_t stride,
                                                                const void *__restrict__ gamma, int weight_type,
                                                                const float2 *__restrict__ stats,
                                                                const T *__restrict__ grads, int64_t grads_stride,
                                                                int64_t n, int64_t c, T *__restrict__ d_feats)
{
    __shared__ float scratch[kWaves];
    for (int64_t row = blockIdx.x; row < n; row += gridDim.x) {
        const T *x = feats + row * stride, *g = grads + row * grads_stride;
        const float2 stat = stats[row];
        float a[1], b[1], sum = 0.0f, dot = 0.0f;
        for (int64_t col = threadIdx.x; col < c; col += kThreads) {
            pccnn_load<1>(x + col, a);
            pccnn_load<1>(g + col, b);
            const float s = b[0] * pccnn_element(gamma, weight_type, col);
            sum += s;
            dot = fmaf(s, (a[0] - stat.x) * stat.y, dot);
        }
        sum = block_sum(sum, scratch) / (float)c;
        dot = block_sum(dot, scratch) / (float)c;
        for (int64_t col = threadIdx.x; col < c; col += kThreads) {
            pccnn_load<1>(x + col, a);
            pccnn_load<1>(g + col, b);
            const float s = b[0] * pccnn_element(gamma, weight_type, col);
            b[0] = stat.y * (s - sum - (a[0] - stat.x) * stat.y * dot);
            pccnn_store<1>(d_feats + row * c + col, b);
        }
    }
}

// Column sums of long rows: workgroup (x, y) adds 256 columns over every gridDim.y-th row.
template <typename T>
__global__ __launch_bounds__(kThreads) void norm_columns_wide_kernel(const T *__restrict__ feats, int64_t stride,
                                                                    const float2 *__restrict__ stats,
                                                                    const T *__restrict__ grads, int64_t grads_stride,
                                                                    int64_t n, int64_t c, float *__restrict__ partial)
{
    const int64_t col = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (col >= c) return;
    float dg = 0.0f, db = 0.0f, a[1], b[1];
    for (int64_t row = blockIdx.y; row < n; row += gridDim.y) {
        const float2 stat = stats[row];
        pccnn_load<1>(feats + row * stride + col, a);
        pccnn_load<1>(grads + row * grads_stride + col, b);
        dg = fmaf(b[0], (a[0] - stat.x) * stat.y, dg);
        db += b[0];
    }
    partial[((int64_t)blockIdx.y * 2) * c + col] = dg;
    partial[((int64_t)blockIdx.y * 2 + 1) * c + col] = db;
}

// Sum over the parts, in order: 16 columns of the [parts][2 c] table per workgroup, 64 threads to a column.
constexpr int kReduceThreads = 1024, kReduceColumns = 16;
__global__ __launch_bounds__(kReduceThreads) void norm_reduce_kernel(const float *__restrict__ partial, int parts,
                                                                    int64_t c, void *__restrict__ d_gamma,
                                                                    void *__restrict__ d_beta, int weight_type)
{
    constexpr int GROUPS = kReduceThreads / kReduceColumns;
    __shared__ float sums[GROUPS][kReduceColumns];
    const int64_t col = (int64_t)blockIdx.x * kReduceColumns + threadIdx.x % kReduceColumns;
    const int group = threadIdx.x / kReduceColumns;
    float total = 0.0f;
    if (col < 2 * c) {
        float x[8];
        int p = group;
        for (; p + 7 * GROUPS < parts; p += 8 * GROUPS) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = partial[(int64_t)(p + i * GROUPS) * 2 * c + col];
#pragma unroll
            for (int i = 0; i < 8; ++i) total += x[i];
        }
        for (; p < parts; p += GROUPS) total += partial[(int64_t)p * 2 * c + col];
    }
    sums[group][threadIdx.x % kReduceColumns] = total;
    __syncthreads();
    if (threadIdx.x >= kReduceColumns || col >= 2 * c) return;
    total = 0.0f;
#pragma unroll 8
    for (int g = 0; g < GROUPS; ++g) total += sums[g][threadIdx.x];
    if (col < c)
        pccnn_set_element(d_gamma, weight_type, col, total);
    else
        pccnn_set_element(d_beta, weight_type, col - c, total);
}

// How a row of c values is laid over lanes: VEC values per load (16 bytes when every row allows it), the fewest lanes of
// 8 .. 64 that hold the row in one load each, then more loads per lane.
struct NormShape {
    int vec, lanes, chunks;
};
NormShape norm_shape(int64_t c, int type, int align)
{
    NormShape s;
    const int full = 16 / pccnn_type_bytes(type);
    s.vec = align == 16 && c % full == 0 ? full : (type == PCCNN_TYPE_BF16 && align >= 4 && c % 2 == 0 ? 2 : 1);
    const int64_t units = pccnn_ceil_div(c, s.vec);
    s.lanes = units <= 8 ? 8 : units <= 16 ? 16 : units <= 32 ? 32 : 64;
    s.chunks = 1;
    while ((int64_t)s.lanes * s.chunks < units) s.chunks *= 2;
    return s;
}
// The widest alignment (16, 4 or 1 bytes) that every row of a call's tensors has.
int norm_align(int64_t c, int type, const void *a, int64_t a_stride, const void *b, int64_t b_stride, const void *d)
{
    for (int bytes = 16; bytes > 1; bytes /= 4)
        if (pccnn_rows_aligned(a, a_stride, type, bytes) && pccnn_rows_aligned(b, b_stride, type, bytes) &&
            pccnn_rows_aligned(d, c, type, bytes))
            return bytes;
    return 1;
}
// Rows that fit a wavefront's registers at their load width.
bool norm_in_registers(const NormShape &s) { return s.vec * s.chunks <= kRegisterColumns / PCCNN_WAVE && s.chunks <= kMostLoads; }

unsigned norm_blocks(int64_t n, int lanes, int waves, int most)
{
    const int64_t rows = (int64_t)waves * (PCCNN_WAVE / lanes);
    return (unsigned)std::max<int64_t>(1, std::min<int64_t>(most, pccnn_ceil_div(n, rows)));
}

// Few rows stay in one workgroup, which needs no second kernel for its sums when it can write them as they are (f32).  It may
// pass over its rows as often as that costs less than the second launch (backward pass, two kernels -> one, f32): 32 rows of
// 64 values 4.9 -> 2.8 us, 128 of 64 5.0 -> 3.8, 16 of 1024 7.3 -> 5.9; four passes over rows of 1024 (7.3 -> 8.4) or two over
// rows of 1021 single values in bf16 (8.2 -> 8.8) would lose.
unsigned norm_back_blocks(int64_t n, const NormShape &s, bool alone)
{
    const int64_t passes = s.chunks == 1 ? 4 : s.chunks <= 4 ? 2 : 1;
    if (alone && n <= passes * kBackWaves * (PCCNN_WAVE / s.lanes)) return 1;
    return norm_blocks(n, s.lanes, kBackWaves, kBackBlocks);
}

// Rows of column sums that a backward pass leaves: of long rows, and at most (long rows that do not fit registers only for
// their loads' width, from 1025 values on, leave 204 or fewer).
int64_t norm_wide_parts(int64_t n, int64_t c)
{
    return std::min(n, std::max<int64_t>(1, kMaxBlocks / pccnn_ceil_div(c, kThreads)));
}
int64_t norm_most_parts(int64_t n, int64_t c)
{
    return c <= kRegisterColumns ? std::min<int64_t>(n, kBackBlocks) : norm_wide_parts(n, c);
}

struct NormForward {
    const void *feats;
    int64_t stride;
    const void *gamma, *beta;
    int weight_type;
    float eps;
    int64_t n, c;
    void *out;
    float *stats;
    hipStream_t stream;
    template <typename T, int VEC, int LANES, int CHUNKS> void launch() const
    {
        norm_fwd_kernel<T, VEC, LANES, CHUNKS><<<norm_blocks(n, LANES, kWaves, kMaxBlocks), kThreads, 0, stream>>>(
            (const T *)feats, stride, gamma, beta, weight_type, eps, n, (int)c, (T *)out, (float2 *)stats);
    }
};
struct NormBackward {
    const void *feats;
    int64_t stride;
    const void *gamma;
    int weight_type;
    const float *stats;
    const void *grads;
    int64_t grads_stride, n, c;
    void *d_feats;
    float *sums_gamma, *sums_beta;
    int64_t sums_stride;
    unsigned blocks;
    hipStream_t stream;
    template <typename T, int VEC, int LANES, int CHUNKS> void launch() const
    {
        norm_bwd_kernel<T, VEC, LANES, CHUNKS><<<blocks, kBackThreads, 0, stream>>>(
            (const T *)feats, stride, gamma, weight_type, (const float2 *)stats, (const T *)grads, grads_stride, n, (int)c,
            (T *)d_feats, sums_gamma, sums_beta, sums_stride);
    }
};
template <typename T, int VEC, typename CALL> void norm_launch_shape(const NormShape &s, const CALL &call)
{
    if (s.lanes == 8) return call.template launch<T, VEC, 8, 1>();
    if (s.lanes == 16) return call.template launch<T, VEC, 16, 1>();
    if (s.lanes == 32) return call.template launch<T, VEC, 32, 1>();
    if (s.chunks == 1) return call.template launch<T, VEC, 64, 1>();
    if (s.chunks == 2) return call.template launch<T, VEC, 64, 2>();
    if (s.chunks == 4) return call.template launch<T, VEC, 64, 4>();
    if constexpr (VEC <= 4) {
        if (s.chunks == 8) return call.template launch<T, VEC, 64, 8>();
        if constexpr (VEC <= 2) return call.template launch<T, VEC, 64, 16>();
    }
}
template <typename CALL> void norm_launch(const NormShape &s, int type, const CALL &call)
{
    if (type == PCCNN_TYPE_F32) {
        if (s.vec == 4) return norm_launch_shape<float, 4>(s, call);
        return norm_launch_shape<float, 1>(s, call);
    }
    if (s.vec == 8) return norm_launch_shape<uint16_t, 8>(s, call);
    if (s.vec == 2) return norm_launch_shape<uint16_t, 2>(s, call);
    return norm_launch_shape<uint16_t, 1>(s, call);
}

int norm_check(const char *name, int type, int weight_type, int64_t n, int64_t c, int64_t stride)
{
    PCCNN_REQUIRE(pccnn_type_ok(type) && pccnn_type_ok(weight_type), PCCNN_ERR_UNSUPPORTED,
                  "%s: element types %d, %d (f32 and bf16 only)", name, type, weight_type);
    PCCNN_REQUIRE(n >= 0 && c >= 1 && c <= INT32_MAX / 4 && stride >= 0, PCCNN_ERR_INVALID,
                  "%s: n=%lld, channels=%lld, row stride %lld", name, (long long)n, (long long)c, (long long)stride);
    return PCCNN_OK;
}

} // namespace

extern "C" size_t pccnn_layer_norm_workspace_bytes(int64_t n, int64_t channels)
{
    if (n <= 0 || channels <= 0) return 256;
    return pccnn_align((size_t)norm_most_parts(n, channels) * 2 * (size_t)channels * sizeof(float));
}

extern "C" int pccnn_layer_norm_forward(const void *feats, int type, int64_t row_stride, const void *gamma,
                                        const void *beta, int weight_type, float eps, int64_t n, int64_t channels,
                                        void *out, float *stats_out, void *stream)
{
    const int rc = norm_check("layer_norm", type, weight_type, n, channels, row_stride);
    if (rc != PCCNN_OK) return rc;
    PCCNN_REQUIRE(eps >= 0.0f, PCCNN_ERR_INVALID, "layer_norm: eps=%g", (double)eps);
    if (n == 0) return PCCNN_OK;
    PCCNN_REQUIRE(feats && gamma && beta && out, PCCNN_ERR_INVALID, "layer_norm: null pointer");
    const int align = norm_align(channels, type, feats, row_stride, out, channels, out);
    const NormShape s = norm_shape(channels, type, align);
    const hipStream_t str = (hipStream_t)stream;
    if (norm_in_registers(s)) {
        norm_launch(s, type, NormForward{feats, row_stride, gamma, beta, weight_type, eps, n, channels, out, stats_out, str});
    } else {
        const unsigned blocks = (unsigned)std::min<int64_t>(n, 16384);
        if (type == PCCNN_TYPE_F32)
            norm_fwd_wide_kernel<float><<<blocks, kThreads, 0, str>>>((const float *)feats, row_stride, gamma, beta,
                                                                     weight_type, eps, n, channels, (float *)out,
                                                                     (float2 *)stats_out);
        else
            norm_fwd_wide_kernel<uint16_t><<<blocks, kThreads, 0, str>>>((const uint16_t *)feats, row_stride, gamma, beta,
                                                                        weight_type, eps, n, channels, (uint16_t *)out,
                                                                        (float2 *)stats_out);
    }
    PCCNN_LAUNCH_CHECK();
    return PCCNN_OK;
}

extern "C" int pccnn_layer_norm_backward(const void *feats, int type, int64_t row_stride, const void *gamma,
                                         int weight_type, const float *stats, const void *in_grads,
                                         int64_t grads_stride, int64_t n, int64_t channels, void *d_feats, void *d_gamma,
                                         void *d_beta, void *workspace, size_t workspace_bytes, void *stream)
{
    const int rc = norm_check("layer_norm_grads", type, weight_type, n, channels, std::min(row_stride, grads_stride));
    if (rc != PCCNN_OK) return rc;
    const bool columns = d_gamma != nullptr || d_beta != nullptr;
    PCCNN_REQUIRE(!columns || (d_gamma && d_beta), PCCNN_ERR_INVALID,
                  "layer_norm_grads: the gradients of gamma and beta come together");
    if (!columns && (d_feats == nullptr || n == 0)) return PCCNN_OK;
    PCCNN_REQUIRE(gamma && (n == 0 || (feats && stats && in_grads)), PCCNN_ERR_INVALID, "layer_norm_grads: null pointer");
    float *partial = nullptr;
    if (columns && n > 0) {
        PccnnArena arena(workspace, workspace_bytes);
        partial = arena.take<float>((size_t)norm_most_parts(n, channels) * 2 * (size_t)channels);
        PCCNN_REQUIRE(arena.ok(), PCCNN_ERR_WORKSPACE, "layer_norm_grads: workspace of %zu bytes is too small",
                      workspace_bytes);
    }
    const hipStream_t str = (hipStream_t)stream;
    int parts = 0;
    bool summed = false;
    if (n > 0) {
        const void *written = d_feats != nullptr ? d_feats : feats;
        const int align = norm_align(channels, type, feats, row_stride, in_grads, grads_stride, written);
        const NormShape s = norm_shape(channels, type, align);
        if (norm_in_registers(s)) {
            const bool alone = columns && weight_type == PCCNN_TYPE_F32;
            parts = (int)norm_back_blocks(n, s, alone);
            summed = alone && parts == 1;
            float *sums_gamma = summed ? (float *)d_gamma : partial;
            float *sums_beta = summed ? (float *)d_beta : partial == nullptr ? nullptr : partial + channels;
            norm_launch(s, type, NormBackward{feats, row_stride, gamma, weight_type, stats, in_grads, grads_stride, n,
                                              channels, d_feats, sums_gamma, sums_beta, 2 * channels, (unsigned)parts,
                                              str});
        } else {
            const unsigned blocks = (unsigned)std::min<int64_t>(n, 16384);
            parts = (int)norm_wide_parts(n, channels);
            const dim3 grid((unsigned)pccnn_ceil_div(channels, kThreads), (unsigned)parts);
            auto wide = [&](auto zero) {
                using T = decltype(zero);
                if (d_feats != nullptr)
                    norm_bwd_wide_kernel<T><<<blocks, kThreads, 0, str>>>((const T *)feats, row_stride, gamma, weight_type,
                                                                         (const float2 *)stats, (const T *)in_grads,
                                                                         grads_stride, n, channels, (T *)d_feats);
                if (partial != nullptr)
                    norm_columns_wide_kernel<T><<<grid, kThreads, 0, str>>>((const T *)feats, row_stride,
                                                                           (const float2 *)stats, (const T *)in_grads,
                                                                           grads_stride, n, channels, partial);
            };
            if (type == PCCNN_TYPE_F32)
                wide(0.0f);
            else
                wide((uint16_t)0);
        }
        PCCNN_LAUNCH_CHECK();
    }
    if (columns && !summed) {
        norm_reduce_kernel<<<(unsigned)pccnn_ceil_div(2 * channels, kReduceColumns), kReduceThreads, 0, str>>>(
            partial, parts, channels, d_gamma, d_beta, weight_type);
        PCCNN_LAUNCH_CHECK();
    }
    return PCCNN_OK;
}
