// Rotary positions over several axes: pairs of a head's features turned by angles that depend on the point's position.
//
//   angle[n, p] = pts[n, axes[p]] freqs[p]        (a, b) -> (a cos - b sin, b cos + a sin)
//
// Pair p is (p, p + pairs) of the head's features, or (2p, 2p + 1) in the adjacent layout; features from 2 * pairs on are
// copied.  The gradient of the features is the turn by the negative angle.  A point's cosines and sines are the same
// for all of its heads: a workgroup computes them once for a tile of points into LDS and then streams the tile's features
// through 16-byte loads and stores, so the kernel is bound by HBM: 119997 points of 8 heads of 64 bf16 values 48 us = 5.1
// TB/s, a copy's rate (61 us with tiles of 4096 units, whose angles kept the memory waiting, and with divisions where a
// multiplication serves now); 2048 points of 4 heads of 32 f32 values 2.8 us.  The angle is formed in f64 and reduced to its
// fraction of a turn there: coordinates are not small numbers, and an f32 product of a position of 10^4 and a frequency of
// 1 would already be off by 10^-3.  Gradients of the positions come from the turned features (d angle = b' a_g - ...),
// summed per point by one wavefront with a lane per pair and loads of single values: 119997 points of 8 heads of 64, all turned,
// 71 us in bf16 (3.5 TB/s) and 115 in f32 (4.3); with 16 pairs in a head, a quarter of the lanes at work, 75 and 70.  Features
// that are not turned are copied value by value: the same points with 16 pairs take 149 us in f32 where 32 take 90, 45 and 39 in
// bf16.
#include "elements.h"

#include <algorithm>

namespace {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 4096;              // cosines and sines of one point: 32 KiB of LDS

__device__ __forceinline__ float2 turn_of(float position, float freq)
{
    const double turns = (double)position * (double)freq * 0.15915494309189535;           // 1 / (2 pi)
    const float part = (float)(turns - rint(turns));                                       // -1/2 .. 1/2; NaN, inf -> NaN
    float2 r;
    sincospif(2.0f * part, &r.y, &r.x);
    return r;
}

struct RotaryShape {
    int64_t n;
    int64_t stride_n, stride_h;              // of the input, in elements; the output is dense
    int heads, width, pairs, axes;
    int tile;                                // points per workgroup
    int turned, units;                       // units of work per head: of 2 PV turned features, and with the rest
    uint32_t by_units, by_heads, by_pairs;   // ceil(2^32 / divisor): a quotient by one multiplication (0: divide)
};

__device__ __forceinline__ int quotient(int value, int divisor, uint32_t inverse)
{
    return inverse != 0 ? (int)__umulhi((uint32_t)value, inverse) : value / divisor;
}

template <typename T, int PV, bool ADJACENT>
__global__ __launch_bounds__(kThreads) void rotary_kernel(const T *__restrict__ in, const float *__restrict__ pts,
                                                         const float *__restrict__ freqs, const int *__restrict__ axis_of,
                                                         RotaryShape s, float sign, T *__restrict__ out)
{
    extern __shared__ float2 turns[];        // [tile][pairs]
    const int64_t first = (int64_t)blockIdx.x * s.tile;
    const int points = (int)min((int64_t)s.tile, s.n - first);
    for (int i = threadIdx.x; i < points * s.pairs; i += kThreads) {
        const int point = quotient(i, s.pairs, s.by_pairs), p = i - point * s.pairs;
        const int axis = max(0, min(axis_of[p], s.axes - 1));
        float2 t = turn_of(pts[(first + point) * s.axes + axis], freqs[p]);
        t.y *= sign;
        turns[i] = t;
    }
    __syncthreads();
    const int total = points * s.heads * s.units;
#pragma unroll 2
    for (int u = threadIdx.x; u < total; u += kThreads) {
        const int row = quotient(u, s.units, s.by_units), unit = u - row * s.units;
        const int point = quotient(row, s.heads, s.by_heads), head = row - point * s.heads;
        const T *src = in + (first + point) * s.stride_n + head * s.stride_h;
        T *dst = out + ((first + point) * s.heads + head) * (int64_t)s.width;
        if (unit < s.turned) {
            const int lo = ADJACENT ? 2 * PV * unit : PV * unit;
            const int hi = ADJACENT ? lo + PV : lo + s.pairs;
            const float2 *t = turns + point * s.pairs + PV * unit;
            float a[PV], b[PV], x[PV], y[PV];
            pccnn_load<PV>(src + lo, a);
            pccnn_load<PV>(src + hi, b);
            if constexpr (ADJACENT) {
                if constexpr (PV == 1) {
                    x[0] = a[0] * t[0].x - b[0] * t[0].y;
                    y[0] = b[0] * t[0].x + a[0] * t[0].y;
                } else {
#pragma unroll
                    for (int i = 0; i < PV / 2; ++i) {
                        x[2 * i] = a[2 * i] * t[i].x - a[2 * i + 1] * t[i].y;
                        x[2 * i + 1] = a[2 * i + 1] * t[i].x + a[2 * i] * t[i].y;
                        y[2 * i] = b[2 * i] * t[i + PV / 2].x - b[2 * i + 1] * t[i + PV / 2].y;
                        y[2 * i + 1] = b[2 * i + 1] * t[i + PV / 2].x + b[2 * i] * t[i + PV / 2].y;
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < PV; ++i) {
                    x[i] = a[i] * t[i].x - b[i] * t[i].y;
                    y[i] = b[i] * t[i].x + a[i] * t[i].y;
                }
            }
            pccnn_store<PV>(dst + lo, x);
            pccnn_store<PV>(dst + hi, y);
        } else {
            int col = 2 * s.pairs + (unit - s.turned) * PV;
            for (const int end = min(col + PV, s.width); col < end; ++col) dst[col] = src[col];
        }
    }
}

// d pts[n, a] = sum over the pairs of axis a and the heads of freq (g_b a' - g_a b'), (a', b') the turned pair: the
// derivative of the turn by its angle is (a', b') -> (-b', a').  One wavefront per point, a lane per pair.
template <typename T, bool ADJACENT>
__global__ __launch_bounds__(kThreads) void rotary_points_kernel(const T *__restrict__ in, const float *__restrict__ pts,
                                                                const float *__restrict__ freqs,
                                                                const int *__restrict__ axis_of, RotaryShape s,
                                                                const T *__restrict__ grads, int64_t grads_n,
                                                                int64_t grads_h, float *__restrict__ d_pts)
{
    const int64_t point = (int64_t)blockIdx.x * (kThreads / PCCNN_WAVE) + threadIdx.x / PCCNN_WAVE;
    if (point >= s.n) return;
    float sums[PCCNN_MAX_DIMS];
#pragma unroll
    for (int a = 0; a < PCCNN_MAX_DIMS; ++a) sums[a] = 0.0f;
    for (int p = threadIdx.x % PCCNN_WAVE; p < s.pairs; p += PCCNN_WAVE) {
        const int axis = max(0, min(axis_of[p], s.axes - 1));
        const float2 t = turn_of(pts[point * s.axes + axis], freqs[p]);
        const int lo = ADJACENT ? 2 * p : p, hi = ADJACENT ? 2 * p + 1 : p + s.pairs;
        float total = 0.0f;
        for (int h = 0; h < s.heads; ++h) {
            const T *src = in + point * s.stride_n + h * s.stride_h, *g = grads + point * grads_n + h * grads_h;
            float a[1], b[1], ga[1], gb[1];
            pccnn_load<1>(src + lo, a);
            pccnn_load<1>(src + hi, b);
            pccnn_load<1>(g + lo, ga);
            pccnn_load<1>(g + hi, gb);
            total += gb[0] * (a[0] * t.x - b[0] * t.y) - ga[0] * (b[0] * t.x + a[0] * t.y);
        }
#pragma unroll
        for (int a = 0; a < PCCNN_MAX_DIMS; ++a)
            if (a == axis) sums[a] = fmaf(total, freqs[p], sums[a]);
    }
#pragma unroll
    for (int a = 0; a < PCCNN_MAX_DIMS; ++a) {
        const float total = pccnn_group_sum<PCCNN_WAVE>(sums[a]);
        if (a < s.axes && threadIdx.x % PCCNN_WAVE == 0) d_pts[point * s.axes + a] = total;
    }
}

int rotary_check(const char *name, int type, int64_t n, int heads, int width, int pairs, int axes, int64_t stride_n,
                 int64_t stride_h)
{
    PCCNN_REQUIRE(pccnn_type_ok(type), PCCNN_ERR_UNSUPPORTED, "%s: element type %d (f32 and bf16 only)", name, type);
    PCCNN_REQUIRE(n >= 0 && heads >= 1 && width >= 1 && pairs >= 0 && 2 * (int64_t)pairs <= width && stride_n >= 0 &&
                      stride_h >= 0,
                  PCCNN_ERR_INVALID, "%s: n=%lld, heads=%d, width=%d, pairs=%d, strides %lld, %lld", name, (long long)n,
                  heads, width, pairs, (long long)stride_n, (long long)stride_h);
    PCCNN_REQUIRE(axes >= 1 && axes <= PCCNN_MAX_DIMS && pairs <= kMaxPairs && (int64_t)heads * width <= INT32_MAX / 8,
                  PCCNN_ERR_UNSUPPORTED, "%s: %d axes (1 to %d), %d pairs (up to %d), %d heads of %d features", name, axes,
                  PCCNN_MAX_DIMS, pairs, kMaxPairs, heads, width);
    return PCCNN_OK;
}

template <typename T, int PV> void rotary_launch(const RotaryShape &shape, const T *in, const float *pts,
                                                 const float *freqs, const int *axis_of, int adjacent, float sign, T *out,
                                                 hipStream_t stream)
{
    RotaryShape s = shape;
    s.turned = s.pairs / PV;
    s.units = s.turned + (int)pccnn_ceil_div(s.width - 2 * s.pairs, PV);
    // a workgroup's points: about 1024 units of work (four per thread, so that the angles of some workgroups are formed
    // while others stream) and up to 32 KiB of angles, fewer while that leaves CUs without work
    const int64_t per_point = (int64_t)s.heads * s.units;
    int64_t tile = std::max<int64_t>(1, 1024 / per_point);
    tile = std::min<int64_t>(tile, std::max(1, kMaxPairs / std::max(1, s.pairs)));
    tile = std::min<int64_t>(tile, std::max<int64_t>(1, pccnn_ceil_div(s.n, 1024)));
    s.tile = (int)tile;
    // value * inverse / 2^32 is the quotient while value * divisor < 2^32 (the inverse is less than one too large)
    auto inverse = [&](int64_t largest, int64_t divisor) -> uint32_t {
        return divisor > 1 && largest * divisor < (1ll << 32) ? (uint32_t)pccnn_ceil_div(1ll << 32, divisor) : 0;
    };
    s.by_units = inverse(tile * per_point, s.units);
    s.by_heads = inverse(tile * s.heads, s.heads);
    s.by_pairs = inverse(tile * s.pairs, s.pairs);
    const unsigned blocks = (unsigned)pccnn_ceil_div(s.n, tile);
    const size_t lds = (size_t)tile * s.pairs * sizeof(float2);
    if (adjacent)
        rotary_kernel<T, PV, true><<<blocks, kThreads, lds, stream>>>(in, pts, freqs, axis_of, s, sign, out);
    else
        rotary_kernel<T, PV, false><<<blocks, kThreads, lds, stream>>>(in, pts, freqs, axis_of, s, sign, out);
}

template <typename T> int rotary_run(const RotaryShape &s, int type, const void *in, const float *pts, const float *freqs,
                                     const int *axis_of, int adjacent, float sign, void *out, hipStream_t stream)
{
    // the widest load (16 or 8 bytes, else single values) that both halves of every pair's run start at a multiple of
    auto fits = [&](int count) {
        const int bytes = count * pccnn_type_bytes(type);
        return s.pairs % count == 0 && s.width % count == 0 && pccnn_rows_aligned(in, s.stride_n, type, bytes) &&
               pccnn_rows_aligned(in, s.stride_h, type, bytes) && pccnn_rows_aligned(out, s.width, type, bytes);
    };
    constexpr int FULL = 16 / (int)sizeof(T);
    if (fits(FULL))
        rotary_launch<T, FULL>(s, (const T *)in, pts, freqs, axis_of, adjacent, sign, (T *)out, stream);
    else if (fits(FULL / 2))
        rotary_launch<T, FULL / 2>(s, (const T *)in, pts, freqs, axis_of, adjacent, sign, (T *)out, stream);
    else
        rotary_launch<T, 1>(s, (const T *)in, pts, freqs, axis_of, adjacent, sign, (T *)out, stream);
    PCCNN_LAUNCH_CHECK();
    return PCCNN_OK;
}

} // namespace

extern "C" int pccnn_rotary(const void *feats, int type, int64_t stride_n, int64_t stride_h, const float *pts,
                            const float *freqs, const int32_t *axes, int64_t n, int heads, int width, int pairs,
                            int num_axes, int adjacent, int backwards, void *out, void *stream)
{
    const int rc = rotary_check("rotary", type, n, heads, width, pairs, num_axes, stride_n, stride_h);
    if (rc != PCCNN_OK) return rc;
    if (n == 0) return PCCNN_OK;
    PCCNN_REQUIRE(feats && pts && out && (pairs == 0 || (freqs && axes)), PCCNN_ERR_INVALID, "rotary: null pointer");
    PCCNN_REQUIRE(n <= (int64_t)INT32_MAX, PCCNN_ERR_UNSUPPORTED, "rotary: n=%lld (up to 2^31 - 1)", (long long)n);
    const RotaryShape s = {n, stride_n, stride_h, heads, width, pairs, num_axes, 0, 0, 0, 0, 0, 0};
    const float sign = backwards ? -1.0f : 1.0f;
    const hipStream_t str = (hipStream_t)stream;
    if (type == PCCNN_TYPE_F32) return rotary_run<float>(s, type, feats, pts, freqs, axes, adjacent, sign, out, str);
    return rotary_run<uint16_t>(s, type, feats, pts, freqs, axes, adjacent, sign, out, str);
}

extern "C" int pccnn_rotary_points_backward(const void *feats, int type, int64_t stride_n, int64_t stride_h,
                                            const float *pts, const float *freqs, const int32_t *axes,
                                            const void *in_grads, int64_t grads_stride_n, int64_t grads_stride_h, int64_t n,
                                            int heads, int width, int pairs, int num_axes, int adjacent, float *d_pts,
                                            void *stream)
{
    const int rc = rotary_check("rotary_grads", type, n, heads, width, pairs, num_axes, std::min(stride_n, grads_stride_n),
                                std::min(stride_h, grads_stride_h));
    if (rc != PCCNN_OK) return rc;
    if (n == 0) return PCCNN_OK;
    PCCNN_REQUIRE(feats && pts && in_grads && d_pts && (pairs == 0 || (freqs && axes)), PCCNN_ERR_INVALID,
                  "rotary_grads: null pointer");
    PCCNN_REQUIRE(n <= (int64_t)INT32_MAX, PCCNN_ERR_UNSUPPORTED, "rotary_grads: n=%lld (up to 2^31 - 1)", (long long)n);
    const RotaryShape s = {n, stride_n, stride_h, heads, width, pairs, num_axes, 0, 0, 0, 0, 0, 0};
    const unsigned blocks = (unsigned)pccnn_ceil_div(n, kThreads / PCCNN_WAVE);
    const hipStream_t str = (hipStream_t)stream;
    auto run = [&](auto zero) {
        using T = decltype(zero);
        if (adjacent)
            rotary_points_kernel<T, true><<<blocks, kThreads, 0, str>>>((const T *)feats, pts, freqs, axes, s,
                                                                      (const T *)in_grads, grads_stride_n, grads_stride_h,
                                                                      d_pts);
        else
            rotary_points_kernel<T, false><<<blocks, kThreads, 0, str>>>((const T *)feats, pts, freqs, axes, s,
                                                                       (const T *)in_grads, grads_stride_n,
                                                                       grads_stride_h, d_pts);
    };
    if (type == PCCNN_TYPE_F32)
        run(0.0f);
    else
        run((uint16_t)0);
    PCCNN_LAUNCH_CHECK();
    return PCCNN_OK;
}
