// Root-mean-square norm of feature rows with the residual's addition in front of it, forward and backward, and rows in 8 bits.
//
//   s = x (+ r, rounded to the type)   rstd = 1 / sqrt(avg(s^2) + eps)   y = s rstd gamma
//   ds = rstd (dy gamma - s rstd^2 avg(dy gamma s)) (+ gradient of s)   dx = dr = ds   dgamma = sum_rows dy s rstd
//   8 bits: t = s gamma   a = max |t|   code = nearest integer of 127 t / a (ties to even)   scale = a rstd / 127
//
// A row lives in the registers of LANES lanes: 8 to 64 of a wavefront (64 / LANES rows at a time), or the 256 of a workgroup;
// it is read once, 16 bytes to a load wherever the row starts.  Rows of more than 8192 values are read again from the
// caches.  The row's factor is common to t and a, so no code depends on a rounding of it; t, a and the quotient are 64 bits
// wide, so codes are the nearest integers, whichever way the row is laid over lanes.
//
// Bound by memory: bf16 65536 x 256 with a residual, forward 25 us and backward 25 + 4 (134 MB each, 5.4 TB/s where a copy of
// 1 GiB has 5.2); 800000 x 128 with a residual to 8 bits 146 us (4.9 TB/s, vector ALU 70 % with the 64-bit quotients); 1037
// rows of 1365 5.5 us; eight rows 2 us, which is a launch.  bf16 rows that are not whole units take longer than their bytes:
// 20000 x 333 with a residual 17 us forward and 25 backward for 10 each (two wavefronts to a SIMD in the backward kernel, each with one
// row on its way, whose end comes in single loads; f32, twice the bytes, 19 and 22), 1000 x 8191 26 and 33 + 8 for 13 each.
#include "elements.h"

#include <algorithm>
#include <float.h>

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / PCCNN_WAVE;
// Six workgroups to a compute unit are there all at once, whatever the registers; of 2048, seven to a unit fit and the rest wait
// (800000 x 128 in 8 bits 153 us, with 2048 171; 65536 x 512 46 and 51).
constexpr int kMaxBlocks = 1536;
constexpr int kBackBlocks = 512;
constexpr int kMostValues = 32;              // of a row, in a lane

// Sum and largest over the LANES lanes that share a row; LANES = 256: over the workgroup, all of whose threads take part.
template <int LANES> __device__ __forceinline__ float row_sum(float v, float *scratch)
{
    if constexpr (LANES <= PCCNN_WAVE) return pccnn_group_sum<LANES>(v);
    v = pccnn_group_sum<PCCNN_WAVE>(v);
    __syncthreads();
    if (threadIdx.x % PCCNN_WAVE == 0) scratch[threadIdx.x / PCCNN_WAVE] = v;
    __syncthreads();
    float total = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) total += scratch[w];
    return total;
}
// Of magnitudes: their bit patterns are ordered like the values, NaN above all.
template <int LANES> __device__ __forceinline__ double row_most(double v, double *scratch)
{
    unsigned long long bits = __double_as_longlong(v);
#pragma unroll
    for (int o = (LANES < PCCNN_WAVE ? LANES : PCCNN_WAVE) / 2; o > 0; o >>= 1) {
        const unsigned long long other = __shfl_xor(bits, o);
        bits = other > bits ? other : bits;
    }
    if constexpr (LANES > PCCNN_WAVE) {
        __syncthreads();
        if (threadIdx.x % PCCNN_WAVE == 0) scratch[threadIdx.x / PCCNN_WAVE] = __longlong_as_double(bits);
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const unsigned long long other = __double_as_longlong(scratch[w]);
            bits = other > bits ? other : bits;
        }
    }
    return __longlong_as_double(bits);
}

// 1 / sqrt(avg + eps) from the sum of squares is `lift` times the result.  lift is 1 but for rows whose squares leave f32: values
// beyond 10^19, or below 10^-19 under an eps below the smallest normal f32 (from which on eps covers what small squares lose: at
// most 2^-150 each).  Their squares are summed again, scaled, by `again`, and the caller takes its values times lift, so that neither
// they nor the result leave f32.
constexpr float kShrink = 0x1p-80f, kGrow = 0x1p100f;
template <typename AGAIN> __device__ __forceinline__ float rstd_of(float squares, float inv_c, float eps, float &lift, AGAIN again)
{
    const float most = squares * inv_c + eps;
    const bool high = !(squares <= FLT_MAX), low = most < FLT_MIN;
    lift = 1.0f;
    if (__any(high || low)) {
        const float scale = high ? kShrink : low ? kGrow : 1.0f;
        const float scaled = again(scale) * inv_c + eps * scale * scale;
        if (high) {
            lift = 0x1p-8f;
            return kShrink / lift / sqrtf(scaled);
        }
        if (low) {
            lift = kGrow;
            return 1.0f / sqrtf(scaled);
        }
    }
    return 1.0f / sqrtf(most);
}

// COUNT codes of 127 t / a: a's reciprocal, the quotient and what it leaves corrected once, which is the correctly rounded
// quotient wherever that is near a border between two integers.  Rows without a finite, positive a: zeros.
__device__ __forceinline__ int code_of(double t, double a, double inv_a)
{
    const double u = 127.0 * t, y = u * inv_a;
    return (int)rint(fma(fma(-a, y, u), inv_a, y));
}

// VEC values (16 bytes) of a row; single values instead took up to twice as long (training 20000 x 333 f32 74 us, 44 so; bf16 88 and
// 43; 8 bits 36 and 20; only bf16 inference of 20000 x 99 7.3 and 8.5).  WHOLE (65536 x 256 bf16 backward 6 us less): every row starts
// at a multiple of 16 bytes and has whole units; else at any address a value may have, and of the last ones only the `left` that
// exist, zeros behind them.  Their addresses are kept from the compiler, which would make one access of what both branches have, and
// two of a whole unit.
template <typename T> __device__ __forceinline__ __attribute__((address_space(1))) T *row_end(T *p)
{
    uint64_t at = (uint64_t)p;
    asm("" : "+v"(at));
    return (__attribute__((address_space(1))) T *)at;
}
template <bool WHOLE, int VEC, typename T> __device__ __forceinline__ void row_load(const T *p, int left, float (&v)[VEC])
{
    static_assert(VEC * sizeof(T) == 16, "16 bytes");
    if constexpr (WHOLE) {
        pccnn_load<VEC>(p, v);
    } else {
        T t[VEC];
        if (left >= VEC) {
            __builtin_memcpy(t, p, 16);
        } else {
            const auto end = row_end(p);
#pragma unroll
            for (int i = 0; i < VEC; ++i) t[i] = i < left ? end[i] : (T)0;
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            if constexpr (std::is_same<T, float>::value)
                v[i] = t[i];
            else
                v[i] = pccnn_bf16_value(t[i]);
    }
}
template <bool WHOLE, int VEC, typename T> __device__ __forceinline__ void row_store(T *p, int left, const float (&v)[VEC])
{
    if constexpr (WHOLE) {
        pccnn_store<VEC>(p, v);
    } else {
        alignas(16) T t[VEC];
        pccnn_store<VEC>(t, v);
        if (left >= VEC) {
            __builtin_memcpy(p, t, 16);
        } else {
            const auto end = row_end(p);
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                if (i < left) end[i] = t[i];
        }
    }
}
template <bool WHOLE, int VEC> __device__ __forceinline__ void row_store_codes(int8_t *p, int left, const int (&q)[VEC])
{
    if (WHOLE || left >= VEC) {
        alignas(8) uint32_t w[VEC / 4];
#pragma unroll
        for (int i = 0; i < VEC / 4; ++i)
            w[i] = (uint32_t)(q[4 * i] & 255) | (uint32_t)(q[4 * i + 1] & 255) << 8 | (uint32_t)(q[4 * i + 2] & 255) << 16 |
                   (uint32_t)q[4 * i + 3] << 24;
        __builtin_memcpy(WHOLE ? __builtin_assume_aligned(p, VEC) : p, w, VEC);
    } else {
        const auto end = row_end(p);
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            if (i < left) end[i] = (int8_t)q[i];
    }
}

struct RmsArgs {
    const void *feats, *residual;            // residual: nullable
    int64_t stride, residual_stride;
    const void *gamma;                       // null: rows as they are (8 bits)
    int weight_type;
    float eps;
    int64_t n, c;
    void *out, *total;
    float *rstd;                             // nullable
    int8_t *codes;
    float *scales;
};

// CODES: the result in 8 bits.
template <typename T, bool CODES, bool WHOLE, int VEC, int LANES, int CHUNKS>
__global__ __launch_bounds__(kThreads) void rms_fwd_kernel(RmsArgs a)
{
    constexpr int ROWS = LANES <= PCCNN_WAVE ? kThreads / LANES : 1;                 // of a workgroup at a time
    __shared__ double scratch[LANES > PCCNN_WAVE ? 2 * kWaves : 1];
    const int lane = threadIdx.x % LANES, slot = threadIdx.x / LANES, c = (int)a.c;
    const float inv_c = 1.0f / (float)c;
    float g[CHUNKS][VEC];
#pragma unroll
    for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const int col = (k * LANES + lane) * VEC + i;
            g[k][i] = a.gamma == nullptr ? 1.0f : col < c ? pccnn_element(a.gamma, a.weight_type, col) : 0.0f;
        }
    for (int64_t base = (int64_t)blockIdx.x * ROWS; base < a.n; base += (int64_t)gridDim.x * ROWS) {
        const int64_t row = base + slot;
        const bool live = row < a.n;
        float x[CHUNKS][VEC], squares = 0.0f;
#pragma unroll
        for (int k = 0; k < CHUNKS; ++k) {
            const int col = (k * LANES + lane) * VEC;
            const bool in = live && col < c;
            if (in) {
                row_load<WHOLE, VEC>((const T *)a.feats + row * a.stride + col, c - col, x[k]);
            } else {
#pragma unroll
                for (int i = 0; i < VEC; ++i) x[k][i] = 0.0f;
            }
            if (a.residual != nullptr && in) {
                float r[VEC];
                row_load<WHOLE, VEC>((const T *)a.residual + row * a.residual_stride + col, c - col, r);
#pragma unroll
                for (int i = 0; i < VEC; ++i) x[k][i] += r[i];
                if constexpr (!std::is_same<T, float>::value) {                      // the stream as it is stored
#pragma unroll
                    for (int i = 0; i < VEC; ++i) x[k][i] = pccnn_bf16_value((uint16_t)pccnn_bf16_pair(x[k][i], x[k][i]));
                }
                row_store<WHOLE, VEC>((T *)a.total + row * a.c + col, c - col, x[k]);
            }
#pragma unroll
            for (int i = 0; i < VEC; ++i) squares = fmaf(x[k][i], x[k][i], squares);
        }
        float rstd = 1.0f;
        if (!CODES || a.gamma != nullptr) {
            squares = row_sum<LANES>(squares, (float *)scratch);
            float lift;
            rstd = rstd_of(squares, inv_c, a.eps, lift, [&](float scale) {
                float again = 0.0f;
#pragma unroll
                for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
                    for (int i = 0; i < VEC; ++i) again = fmaf(x[k][i] * scale, x[k][i] * scale, again);
                return row_sum<LANES>(again, (float *)scratch);
            });
            if (a.rstd != nullptr && live && lane == 0) a.rstd[row] = rstd * lift;
            if (lift != 1.0f) {
#pragma unroll
                for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
                    for (int i = 0; i < VEC; ++i) x[k][i] *= lift;
            }
        }
        if constexpr (CODES) {
            double most = 0.0;
            bool odd = false;
#pragma unroll
            for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const double t = fabs((double)x[k][i] * (double)g[k][i]);
                    odd |= !(t <= DBL_MAX);
                    most = fmax(most, t);
                }
            most = row_most<LANES>(odd ? NAN : most, scratch + (LANES > PCCNN_WAVE ? kWaves : 0));
            const bool fine = most > 0.0 && most <= DBL_MAX;
            const double inv = fine ? 1.0 / most : 0.0;
            if (!live) continue;
            if (lane == 0) a.scales[row] = fine ? (float)(most * (double)rstd / 127.0) : most == 0.0 ? 0.0f : NAN;
#pragma unroll
            for (int k = 0; k < CHUNKS; ++k) {
                const int col = (k * LANES + lane) * VEC;
                if (col >= c) continue;
                int q[VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) q[i] = fine ? code_of((double)x[k][i] * (double)g[k][i], most, inv) : 0;
                row_store_codes<WHOLE, VEC>(a.codes + row * a.c + col, c - col, q);
            }
        } else {
            if (!live) continue;
#pragma unroll
            for (int k = 0; k < CHUNKS; ++k) {
                const int col = (k * LANES + lane) * VEC;
                if (col >= c) continue;
                float y[VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) y[i] = x[k][i] * rstd * g[k][i];
                row_store<WHOLE, VEC>((T *)a.out + row * a.c + col, c - col, y);
            }
        }
    }
}

// Rows of any length: a workgroup per row, read again for every pass over it.
template <typename T, bool CODES> __global__ __launch_bounds__(kThreads) void rms_fwd_wide_kernel(RmsArgs a)
{
    __shared__ double scratch[2 * kWaves];
    for (int64_t row = blockIdx.x; row < a.n; row += gridDim.x) {
        const T *x = (const T *)a.feats + row * a.stride;
        float v[1], r[1], squares = 0.0f;
        double most = 0.0;
        bool odd = false;
        auto weight = [&](int64_t col) { return a.gamma == nullptr ? 1.0f : pccnn_element(a.gamma, a.weight_type, col); };
        for (int64_t col = threadIdx.x; col < a.c; col += kThreads) {
            pccnn_load<1>(x + col, v);
            if (a.residual != nullptr) {
                pccnn_load<1>((const T *)a.residual + row * a.residual_stride + col, r);
                v[0] += r[0];
                if constexpr (!std::is_same<T, float>::value) v[0] = pccnn_bf16_value((uint16_t)pccnn_bf16_pair(v[0], v[0]));
                pccnn_store<1>((T *)a.total + row * a.c + col, v);
            }
            squares = fmaf(v[0], v[0], squares);
            if constexpr (CODES) {
                const double t = fabs((double)v[0] * (double)weight(col));
                odd |= !(t <= DBL_MAX);
                most = fmax(most, t);
            }
        }
        const T *s = a.residual != nullptr ? (const T *)a.total + row * a.c : x;     // (a thread reads what it wrote)
        float rstd = 1.0f, lift = 1.0f;
        if (!CODES || a.gamma != nullptr) {
            squares = row_sum<kThreads>(squares, (float *)scratch);
            rstd = rstd_of(squares, 1.0f / (float)a.c, a.eps, lift, [&](float scale) {
                float again = 0.0f;
                for (int64_t col = threadIdx.x; col < a.c; col += kThreads) {
                    pccnn_load<1>(s + col, v);
                    again = fmaf(v[0] * scale, v[0] * scale, again);
                }
                return row_sum<kThreads>(again, (float *)scratch);
            });
            if (a.rstd != nullptr && threadIdx.x == 0) a.rstd[row] = rstd * lift;
        }
        if constexpr (CODES) most = row_most<kThreads>(odd ? NAN : most, scratch + kWaves);
        const bool fine = most > 0.0 && most <= DBL_MAX;
        if constexpr (CODES) {
            if (threadIdx.x == 0) a.scales[row] = fine ? (float)(most * (double)lift * (double)rstd / 127.0) : most == 0.0 ? 0.0f : NAN;
        }
        const double inv = fine ? 1.0 / most : 0.0;
        for (int64_t col = threadIdx.x; col < a.c; col += kThreads) {
            pccnn_load<1>(s + col, v);
            if constexpr (CODES) {
                a.codes[row * a.c + col] = (int8_t)(fine ? code_of((double)v[0] * (double)weight(col), most, inv) : 0);
            } else {
                v[0] = v[0] * lift * rstd * weight(col);
                pccnn_store<1>((T *)a.out + row * a.c + col, v);
            }
        }
    }
}

// ------------------------------------------------------------------------------------------- backward

struct RmsBackArgs {
    const void *total, *gamma, *grads, *total_grads;      // total_grads: nullable
    int64_t stride, grads_stride, total_grads_stride;
    int weight_type;
    const float *rstd;
    int64_t n, c;
    void *d_feats;                           // nullable
    float *sums;                             // nullable: a row of column sums for each workgroup
};
template <typename T, bool WHOLE, int VEC, int LANES, int CHUNKS>
__global__ __launch_bounds__(kThreads) void rms_bwd_kernel(RmsBackArgs a)
{
    constexpr int ROWS = LANES <= PCCNN_WAVE ? kThreads / LANES : 1, COLUMNS = LANES * CHUNKS * VEC;
    __shared__ float scratch[kWaves];
    __shared__ float sums[LANES <= PCCNN_WAVE ? kWaves : 1][LANES <= PCCNN_WAVE ? COLUMNS : 1];
    const int lane = threadIdx.x % LANES, slot = threadIdx.x / LANES, c = (int)a.c;
    const float inv_c = 1.0f / (float)c;
    float w[CHUNKS][VEC], dg[CHUNKS][VEC];
#pragma unroll
    for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const int col = (k * LANES + lane) * VEC + i;
            w[k][i] = col < c ? pccnn_element(a.gamma, a.weight_type, col) : 0.0f;
            dg[k][i] = 0.0f;
        }
    for (int64_t base = (int64_t)blockIdx.x * ROWS; base < a.n; base += (int64_t)gridDim.x * ROWS) {
        const int64_t row = base + slot;
        const bool live = row < a.n;
        const float rstd = live ? a.rstd[row] : 0.0f;
        float x[CHUNKS][VEC], g[CHUNKS][VEC], dot = 0.0f;
#pragma unroll
        for (int k = 0; k < CHUNKS; ++k) {
            const int col = (k * LANES + lane) * VEC;
            if (live && col < c) {
                row_load<WHOLE, VEC>((const T *)a.total + row * a.stride + col, c - col, x[k]);
                row_load<WHOLE, VEC>((const T *)a.grads + row * a.grads_stride + col, c - col, g[k]);
            } else {
#pragma unroll
                for (int i = 0; i < VEC; ++i) x[k][i] = g[k][i] = 0.0f;
            }
        }
#pragma unroll
        for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                x[k][i] *= rstd;
                dg[k][i] = fmaf(g[k][i], x[k][i], dg[k][i]);
                g[k][i] *= w[k][i];
                dot = fmaf(g[k][i], x[k][i], dot);
            }
        if (a.d_feats == nullptr) continue;
        dot = row_sum<LANES>(dot, scratch) * inv_c;
        if (!live) continue;
#pragma unroll
        for (int k = 0; k < CHUNKS; ++k) {
            const int col = (k * LANES + lane) * VEC;
            if (col >= c) continue;
            float d[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) d[i] = rstd * (g[k][i] - x[k][i] * dot);
            if (a.total_grads != nullptr) {
                float t[VEC];
                row_load<WHOLE, VEC>((const T *)a.total_grads + row * a.total_grads_stride + col, c - col, t);
#pragma unroll
                for (int i = 0; i < VEC; ++i) d[i] += t[i];
            }
            row_store<WHOLE, VEC>((T *)a.d_feats + row * a.c + col, c - col, d);
        }
    }
    if (a.sums == nullptr) return;
    float *mine = a.sums + (int64_t)blockIdx.x * a.c;
    if constexpr (LANES > PCCNN_WAVE) {
#pragma unroll
        for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const int col = (k * LANES + lane) * VEC + i;
                if (col < c) mine[col] = dg[k][i];
            }
    } else {
        const int wave = threadIdx.x / PCCNN_WAVE;
#pragma unroll
        for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float total = pccnn_strided_sum<LANES>(dg[k][i]);
                if (threadIdx.x % PCCNN_WAVE < LANES) sums[wave][(k * LANES + lane) * VEC + i] = total;
            }
        __syncthreads();
        for (int col = threadIdx.x; col < c; col += kThreads) {
            float total = 0.0f;
#pragma unroll
            for (int v = 0; v < kWaves; ++v) total += sums[v][col];
            mine[col] = total;
        }
    }
}

template <typename T> __global__ __launch_bounds__(kThreads) void rms_bwd_wide_kernel(RmsBackArgs a)
{
    __shared__ float scratch[kWaves];
    for (int64_t row = blockIdx.x; row < a.n; row += gridDim.x) {
        const T *x = (const T *)a.total + row * a.stride, *g = (const T *)a.grads + row * a.grads_stride;
        const float rstd = a.rstd[row];
        float v[1], d[1], t[1], dot = 0.0f;
        for (int64_t col = threadIdx.x; col < a.c; col += kThreads) {
            pccnn_load<1>(x + col, v);
            pccnn_load<1>(g + col, d);
            dot = fmaf(d[0] * pccnn_element(a.gamma, a.weight_type, col), v[0] * rstd, dot);
        }
        dot = row_sum<kThreads>(dot, scratch) / (float)a.c;
        for (int64_t col = threadIdx.x; col < a.c; col += kThreads) {
            pccnn_load<1>(x + col, v);
            pccnn_load<1>(g + col, d);
            d[0] = rstd * (d[0] * pccnn_element(a.gamma, a.weight_type, col) - v[0] * rstd * dot);
            if (a.total_grads != nullptr) {
                pccnn_load<1>((const T *)a.total_grads + row * a.total_grads_stride + col, t);
                d[0] += t[0];
            }
            pccnn_store<1>((T *)a.d_feats + row * a.c + col, d);
        }
    }
}
// Column sums of long rows: workgroup (x, y) adds 256 columns over every gridDim.y-th row.
template <typename T> __global__ __launch_bounds__(kThreads) void rms_columns_wide_kernel(RmsBackArgs a)
{
    const int64_t col = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (col >= a.c) return;
    float sum = 0.0f, v[1], g[1];
    for (int64_t row = blockIdx.y; row < a.n; row += gridDim.y) {
        pccnn_load<1>((const T *)a.total + row * a.stride + col, v);
        pccnn_load<1>((const T *)a.grads + row * a.grads_stride + col, g);
        sum = fmaf(g[0], v[0] * a.rstd[row], sum);
    }
    a.sums[(int64_t)blockIdx.y * a.c + col] = sum;
}
// Sum over the parts, in order: 16 columns of the [parts][c] table per workgroup, 64 threads to a column.
constexpr int kReduceThreads = 1024, kReduceColumns = 16;
__global__ __launch_bounds__(kReduceThreads) void rms_reduce_kernel(const float *__restrict__ partial, int parts, int64_t c,
                                                                   void *__restrict__ d_gamma, int weight_type)
{
    constexpr int GROUPS = kReduceThreads / kReduceColumns;
    __shared__ float sums[GROUPS][kReduceColumns];
    const int64_t col = (int64_t)blockIdx.x * kReduceColumns + threadIdx.x % kReduceColumns;
    const int group = threadIdx.x / kReduceColumns;
    float total = 0.0f;
    if (col < c)
#pragma unroll 8
        for (int p = group; p < parts; p += GROUPS) total += partial[(int64_t)p * c + col];
    sums[group][threadIdx.x % kReduceColumns] = total;
    __syncthreads();
    if (threadIdx.x >= kReduceColumns || col >= c) return;
    total = 0.0f;
#pragma unroll 8
    for (int g = 0; g < GROUPS; ++g) total += sums[g][threadIdx.x];
    pccnn_set_element(d_gamma, weight_type, col, total);
}

// ------------------------------------------------------------------------------------------- host

// How a row of c values is laid over lanes: 16 bytes a load, the fewest lanes of 8 .. 64 that hold the row in one load each, then
// more loads per lane, then the lanes of a workgroup.  chunks 0: not in registers.
struct RmsShape {
    int lanes, chunks;
};
RmsShape rms_shape(int64_t c, int type)
{
    const int vec = 16 / pccnn_type_bytes(type), most = kMostValues / vec;
    const int64_t units = pccnn_ceil_div(c, vec);
    RmsShape s = {8, 1};
    while (s.lanes < PCCNN_WAVE && s.lanes < units) s.lanes *= 2;
    if (units > (int64_t)PCCNN_WAVE * 4) s.lanes = kThreads;
    while ((int64_t)s.lanes * s.chunks < units && s.chunks <= most) s.chunks *= 2;
    if (s.chunks > most) s.chunks = 0;
    return s;
}
struct RmsRows {
    const void *p;
    int64_t stride;
};
// Whether every row of a call's tensors has whole 16-byte units at multiples of 16 bytes.
bool rms_whole(int64_t c, int type, std::initializer_list<RmsRows> tensors)
{
    bool all = c * pccnn_type_bytes(type) % 16 == 0;
    for (const RmsRows &t : tensors) all = all && (t.p == nullptr || pccnn_rows_aligned(t.p, t.stride, type, 16));
    return all;
}
int64_t rms_blocks(int64_t n, int lanes, int most)
{
    const int rows = lanes <= PCCNN_WAVE ? kThreads / lanes : 1;
    return std::max<int64_t>(1, std::min<int64_t>(most, pccnn_ceil_div(n, rows)));
}
int64_t rms_wide_parts(int64_t n, int64_t c)
{
    return std::min(n, std::max<int64_t>(1, 1024 / pccnn_ceil_div(c, kThreads)));
}
int64_t rms_most_parts(int64_t n, int64_t c)
{
    return c <= kThreads * kMostValues ? std::min<int64_t>(n, kBackBlocks) : rms_wide_parts(n, c);
}

template <typename T, bool WHOLE, int VEC, typename CALL> void rms_launch_shape(const RmsShape &s, const CALL &call)
{
    if (s.lanes == 8) return call.template launch<T, WHOLE, VEC, 8, 1>();
    if (s.lanes == 16) return call.template launch<T, WHOLE, VEC, 16, 1>();
    if (s.lanes == 32) return call.template launch<T, WHOLE, VEC, 32, 1>();
    if (s.lanes == 64) {
        if (s.chunks == 1) return call.template launch<T, WHOLE, VEC, 64, 1>();
        if (s.chunks == 2) return call.template launch<T, WHOLE, VEC, 64, 2>();
        return call.template launch<T, WHOLE, VEC, 64, 4>();
    }
    if (s.chunks <= 2) return call.template launch<T, WHOLE, VEC, 256, 2>();
    if (s.chunks == 4) return call.template launch<T, WHOLE, VEC, 256, 4>();
    if constexpr (VEC == 4) return call.template launch<T, WHOLE, VEC, 256, 8>();
}
template <typename CALL> void rms_launch(const RmsShape &s, int type, bool whole, const CALL &call)
{
    if (type == PCCNN_TYPE_F32)
        whole ? rms_launch_shape<float, true, 4>(s, call) : rms_launch_shape<float, false, 4>(s, call);
    else
        whole ? rms_launch_shape<uint16_t, true, 8>(s, call) : rms_launch_shape<uint16_t, false, 8>(s, call);
}
template <bool CODES> struct RmsForward {
    const RmsArgs &a;
    hipStream_t stream;
    template <typename T, bool WHOLE, int VEC, int LANES, int CHUNKS> void launch() const
    {
        rms_fwd_kernel<T, CODES, WHOLE, VEC, LANES, CHUNKS><<<(unsigned)rms_blocks(a.n, LANES, kMaxBlocks), kThreads, 0, stream>>>(a);
    }
};
struct RmsBackward {
    const RmsBackArgs &a;
    hipStream_t stream;
    template <typename T, bool WHOLE, int VEC, int LANES, int CHUNKS> void launch() const
    {
        rms_bwd_kernel<T, WHOLE, VEC, LANES, CHUNKS><<<(unsigned)rms_blocks(a.n, LANES, kBackBlocks), kThreads, 0, stream>>>(a);
    }
};

int rms_check(const char *name, int type, int weight_type, int64_t n, int64_t c, int64_t stride)
{
    PCCNN_REQUIRE(pccnn_type_ok(type) && pccnn_type_ok(weight_type), PCCNN_ERR_UNSUPPORTED,
                  "%s: element types %d, %d (f32 and bf16 only)", name, type, weight_type);
    PCCNN_REQUIRE(n >= 0 && c >= 1 && c <= INT32_MAX / 4 && stride >= 0, PCCNN_ERR_INVALID,
                  "%s: n=%lld, channels=%lld, row stride %lld", name, (long long)n, (long long)c, (long long)stride);
    return PCCNN_OK;
}
template <bool CODES> int rms_run(const RmsArgs &a, int type, void *stream)
{
    const hipStream_t s = (hipStream_t)stream;
    const RmsShape shape = rms_shape(a.c, type);
    if (shape.chunks > 0) {
        rms_launch(shape, type, rms_whole(a.c, type, {{a.feats, a.stride}, {a.residual, a.residual_stride}, {a.out, a.c}, {a.total, a.c}}),
                   RmsForward<CODES>{a, s});
    } else {
        const unsigned blocks = (unsigned)std::min<int64_t>(a.n, 16384);
        if (type == PCCNN_TYPE_F32)
            rms_fwd_wide_kernel<float, CODES><<<blocks, kThreads, 0, s>>>(a);
        else
            rms_fwd_wide_kernel<uint16_t, CODES><<<blocks, kThreads, 0, s>>>(a);
    }
    PCCNN_LAUNCH_CHECK();
    return PCCNN_OK;
}

} // namespace

extern "C" size_t pccnn_rms_norm_workspace_bytes(int64_t n, int64_t channels)
{
    if (n <= 0 || channels <= 0 || channels > INT32_MAX / 4) return 256;
    return pccnn_align((size_t)rms_most_parts(n, channels) * (size_t)channels * sizeof(float));
}

extern "C" int pccnn_rms_norm_forward(const void *feats, int type, int64_t row_stride, const void *residual,
                                      int64_t residual_stride, const void *gamma, int weight_type, float eps, int64_t n,
                                      int64_t channels, void *out, void *total_out, float *rstd_out, void *stream)
{
    const int rc = rms_check("rms_norm", type, weight_type, n, channels, std::min(row_stride, residual ? residual_stride : 0));
    if (rc != PCCNN_OK) return rc;
    PCCNN_REQUIRE(eps >= 0.0f, PCCNN_ERR_INVALID, "rms_norm: eps=%g", (double)eps);
    PCCNN_REQUIRE((residual != nullptr) == (total_out != nullptr) || n == 0, PCCNN_ERR_INVALID,
                  "rms_norm: a residual and its sum come together");
    if (n == 0) return PCCNN_OK;
    PCCNN_REQUIRE(feats && gamma && out, PCCNN_ERR_INVALID, "rms_norm: null pointer");
    const RmsArgs a = {feats, residual, row_stride, residual_stride, gamma, weight_type, eps, n, channels, out, total_out,
                       rstd_out, nullptr, nullptr};
    return rms_run<false>(a, type, stream);
}

extern "C" int pccnn_rms_norm_8bit(const void *feats, int type, int64_t row_stride, const void *residual,
                                   int64_t residual_stride, const void *gamma, int weight_type, float eps, int64_t n,
                                   int64_t channels, int8_t *codes_out, float *scales_out, void *total_out, void *stream)
{
    const int rc = rms_check("rms_norm_8bit", type, weight_type, n, channels, std::min(row_stride, residual ? residual_stride : 0));
    if (rc != PCCNN_OK) return rc;
    PCCNN_REQUIRE(eps >= 0.0f, PCCNN_ERR_INVALID, "rms_norm_8bit: eps=%g", (double)eps);
    PCCNN_REQUIRE((residual != nullptr) == (total_out != nullptr) || n == 0, PCCNN_ERR_INVALID,
                  "rms_norm_8bit: a residual and its sum come together");
    if (n == 0) return PCCNN_OK;
    PCCNN_REQUIRE(feats && gamma && codes_out && scales_out, PCCNN_ERR_INVALID, "rms_norm_8bit: null pointer");
    PCCNN_REQUIRE((uintptr_t)codes_out % 16 == 0, PCCNN_ERR_INVALID, "rms_norm_8bit: a result that is not 16-byte aligned");
    const RmsArgs a = {feats, residual, row_stride, residual_stride, gamma, weight_type, eps, n, channels, nullptr, total_out,
                       nullptr, codes_out, scales_out};
    return rms_run<true>(a, type, stream);
}

extern "C" int pccnn_quantize_rows(const void *feats, int type, int64_t row_stride, int64_t n, int64_t channels,
                                   int8_t *codes_out, float *scales_out, void *stream)
{
    const int rc = rms_check("quantize_rows", type, PCCNN_TYPE_F32, n, channels, row_stride);
    if (rc != PCCNN_OK) return rc;
    if (n == 0) return PCCNN_OK;
    PCCNN_REQUIRE(feats && codes_out && scales_out, PCCNN_ERR_INVALID, "quantize_rows: null pointer");
    PCCNN_REQUIRE((uintptr_t)codes_out % 16 == 0, PCCNN_ERR_INVALID, "quantize_rows: a result that is not 16-byte aligned");
    const RmsArgs a = {feats, nullptr, row_stride, 0, nullptr, PCCNN_TYPE_F32, 0.0f, n, channels, nullptr, nullptr, nullptr,
                       codes_out, scales_out};
    return rms_run<true>(a, type, stream);
}

extern "C" int pccnn_rms_norm_backward(const void *total, int type, int64_t row_stride, const void *gamma, int weight_type,
                                       const float *rstd, const void *in_grads, int64_t grads_stride, const void *total_grads,
                                       int64_t total_grads_stride, int64_t n, int64_t channels, void *d_feats, void *d_gamma,
                                       void *workspace, size_t workspace_bytes, void *stream)
{
    const char *name = "rms_norm_grads";
    const int rc = rms_check(name, type, weight_type, n, channels,
                             std::min(std::min(row_stride, grads_stride), total_grads ? total_grads_stride : 0));
    if (rc != PCCNN_OK) return rc;
    if (d_gamma == nullptr && (d_feats == nullptr || n == 0)) return PCCNN_OK;
    PCCNN_REQUIRE(gamma && (n == 0 || (total && rstd && in_grads)), PCCNN_ERR_INVALID, "%s: null pointer", name);
    const hipStream_t s = (hipStream_t)stream;
    RmsBackArgs a = {total, gamma, in_grads, total_grads, row_stride, grads_stride, total_grads_stride, weight_type, rstd, n,
                     channels, d_feats, nullptr};
    int parts = 0;
    if (n > 0) {
        if (d_gamma != nullptr) {
            PccnnArena arena(workspace, workspace_bytes);
            a.sums = arena.take<float>((size_t)rms_most_parts(n, channels) * (size_t)channels);
            PCCNN_REQUIRE(arena.ok(), PCCNN_ERR_WORKSPACE, "%s: workspace of %zu bytes is too small", name, workspace_bytes);
        }
        const RmsShape shape = rms_shape(channels, type);
        if (shape.chunks > 0) {
            parts = (int)rms_blocks(n, shape.lanes, kBackBlocks);
            rms_launch(shape, type,
                       rms_whole(channels, type, {{total, row_stride}, {in_grads, grads_stride}, {total_grads, total_grads_stride},
                                                  {d_feats, channels}}),
                       RmsBackward{a, s});
        } else {
            const unsigned blocks = (unsigned)std::min<int64_t>(n, 16384);
            parts = (int)rms_wide_parts(n, channels);
            const dim3 grid((unsigned)pccnn_ceil_div(channels, kThreads), (unsigned)parts);
            auto wide = [&](auto zero) {
                using T = decltype(zero);
                if (d_feats != nullptr) rms_bwd_wide_kernel<T><<<blocks, kThreads, 0, s>>>(a);
                if (a.sums != nullptr) rms_columns_wide_kernel<T><<<grid, kThreads, 0, s>>>(a);
            };
            if (type == PCCNN_TYPE_F32)
                wide(0.0f);
            else
                wide((uint16_t)0);
        }
        PCCNN_LAUNCH_CHECK();
    }
    if (d_gamma != nullptr) {
        rms_reduce_kernel<<<(unsigned)pccnn_ceil_div(channels, kReduceColumns), kReduceThreads, 0, s>>>(a.sums, parts, channels,
                                                                                                       d_gamma, weight_type);
        PCCNN_LAUNCH_CHECK();
    }
    return PCCNN_OK;
}
