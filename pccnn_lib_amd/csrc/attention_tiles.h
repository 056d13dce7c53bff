// Tiles of the attention kernels: 32 x 32 products on v_mfma_f32_32x32x16_bf16, operands in LDS or registers.
//
// A product C = A B has C's column in the lane (lane & 31) and C's rows 8 (i / 4) + 4 (lane / 32) + i % 4 in its sixteen
// registers i.  A lane's operand of A is eight consecutive k of one row (row = lane & 31, k from 8 (lane / 32)), of B
// eight consecutive k of one column.  Registers 8 g .. 8 g + 7 of C are then, per lane half, the rows
// 16 g + 4 half + {0..3} and 16 g + 8 + 4 half + {0..3}: taken as they are they serve as a B operand of a following product
// over C's rows, if the A operand takes its k in the same order.  The transposing LDS read fetches exactly that order from
// a tile stored row by row, so neither the probabilities nor the tiles are ever moved between lanes.
//
// f32 features are carried as three bf16 terms each (x = x0 + x1 + x2 holds all 24 bits) and a product as the six
// partial products whose terms' indices add up to at most 2; what is left out is below one f32 rounding.
#pragma once
#include "elements.h"

#ifdef __HIPCC__
typedef short pccnn_i16x4 __attribute__((ext_vector_type(4)));
typedef short pccnn_i16x8 __attribute__((ext_vector_type(8)));

template <typename T> struct AttnTerms { static constexpr int value = 3; };
template <> struct AttnTerms<uint16_t> { static constexpr int value = 1; };

// One operand: eight values, as one or three bf16 terms.
template <int TERMS> struct AttnFrag {
    pccnn_bf16x8 t[TERMS];
};

// a and b in three terms each, or a in one and b in one or two.
template <int TERMS, int B> __device__ __forceinline__ void attn_mma(pccnn_f32x16 &c, const AttnFrag<TERMS> &a,
                                                                    const AttnFrag<B> &b)
{
    static_assert(TERMS == B || (TERMS == 1 && B == 2), "");
    if constexpr (TERMS == 3) {                         // smallest products first
        c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.t[2], b.t[0], c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.t[1], b.t[1], c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.t[0], b.t[2], c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.t[1], b.t[0], c, 0, 0, 0);
    }
    if constexpr (B >= 2) c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.t[0], b.t[1], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.t[0], b.t[0], c, 0, 0, 0);
}

// Eight f32 values as terms, each rounded to nearest even from what the terms before it leave.  WHOLE: up to the largest f32
// value, for features (a value within 2^-9 of it would round to an infinite first term; the next terms take what the largest
// finite one leaves).
template <int TERMS, bool WHOLE = false> __device__ __forceinline__ AttnFrag<TERMS> attn_split(const float (&x)[8])
{
    constexpr float most = 0x1.fep127f;                  // of bf16
    AttnFrag<TERMS> f;
    float rest[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) rest[i] = x[i];
#pragma unroll
    for (int t = 0; t < TERMS; ++t) {
        pccnn_u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (WHOLE && t == 0)
                w[i] = pccnn_bf16_pair(__builtin_amdgcn_fmed3f(rest[2 * i], -most, most),
                                       __builtin_amdgcn_fmed3f(rest[2 * i + 1], -most, most));
            else
                w[i] = pccnn_bf16_pair(rest[2 * i], rest[2 * i + 1]);
            if (t + 1 < TERMS) {
                rest[2 * i] -= __uint_as_float(w[i] << 16);
                rest[2 * i + 1] -= __uint_as_float(w[i] & 0xffff0000u);
            }
        }
        f.t[t] = __builtin_bit_cast(pccnn_bf16x8, w);
    }
    return f;
}

// Eight consecutive features of one row, as they lie in memory.
template <typename T> struct AttnChunk;
template <> struct AttnChunk<uint16_t> { pccnn_u32x4 v; };
template <> struct AttnChunk<float> { float v[8]; };

__device__ __forceinline__ void attn_clear(AttnChunk<uint16_t> &c) { c.v = (pccnn_u32x4){0u, 0u, 0u, 0u}; }
__device__ __forceinline__ void attn_clear(AttnChunk<float> &c)
{
#pragma unroll
    for (int i = 0; i < 8; ++i) c.v[i] = 0.0f;
}

// Features col .. col + 7 of a row of `width`, zeros past its end.  `wide`: 2 when width is a multiple of 8 and every row
// starts at a multiple of 16 bytes, 1 when width is a multiple of 4 and rows start at multiples of four elements, else 0.
__device__ __forceinline__ void attn_load(AttnChunk<uint16_t> &c, const uint16_t *row, int col, int width, int wide)
{
    attn_clear(c);
    if (col >= width) return;
    if (wide == 2) {
        c.v = *(const pccnn_u32x4 *)(row + col);
    } else if (wide == 1) {
        const pccnn_u32x2 lo = *(const pccnn_u32x2 *)(row + col);
        c.v[0] = lo[0]; c.v[1] = lo[1];
        if (col + 4 < width) {
            const pccnn_u32x2 hi = *(const pccnn_u32x2 *)(row + col + 4);
            c.v[2] = hi[0]; c.v[3] = hi[1];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (col + i < width) c.v[i / 2] |= (uint32_t)row[col + i] << (16 * (i % 2));
    }
}
__device__ __forceinline__ void attn_load(AttnChunk<float> &c, const float *row, int col, int width, int wide)
{
    attn_clear(c);
    if (col >= width) return;
    if (wide >= 1) {
        const float4 lo = *(const float4 *)(row + col);
        c.v[0] = lo.x; c.v[1] = lo.y; c.v[2] = lo.z; c.v[3] = lo.w;
        if (col + 4 < width) {
            const float4 hi = *(const float4 *)(row + col + 4);
            c.v[4] = hi.x; c.v[5] = hi.y; c.v[6] = hi.z; c.v[7] = hi.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (col + i < width) c.v[i] = row[col + i];
    }
}
// The i-th of a chunk's values.
__device__ __forceinline__ float attn_value(const AttnChunk<uint16_t> &c, int i)
{
    return __uint_as_float(i % 2 ? c.v[i / 2] & 0xffff0000u : c.v[i / 2] << 16);
}
__device__ __forceinline__ float attn_value(const AttnChunk<float> &c, int i) { return c.v[i]; }

__device__ __forceinline__ AttnFrag<1> attn_frag(const AttnChunk<uint16_t> &c)
{
    AttnFrag<1> f;
    f.t[0] = __builtin_bit_cast(pccnn_bf16x8, c.v);
    return f;
}
__device__ __forceinline__ AttnFrag<3> attn_frag(const AttnChunk<float> &c) { return attn_split<3, true>(c.v); }

// A tile of ROWS rows in LDS, bf16, one plane per term, rows of DP features without padding.  The 16-byte units of a row
// are exchanged among themselves by a rule on the row, chosen so that the two reads below touch every group of four banks
// once: sixteen rows at one unit (an operand's rows), and four rows at four neighboring units (its columns).
template <int TERMS, int ROWS, int DP> struct AttnTile {
    static constexpr int UNITS = DP / 8;                              // 16-byte units of a row: 4, 8, 12 or 16
    static constexpr int PLANE = ROWS * DP;                           // elements
    static constexpr int ELEMENTS = TERMS * PLANE;
    uint16_t *base;
    // Where unit `unit` of row `row` lies within the row (its own inverse, except for twelve units).
    static __device__ __forceinline__ int place(int row, int unit)
    {
        if constexpr (UNITS == 4) return unit ^ ((row >> 2) & 3);
        if constexpr (UNITS == 8) return unit ^ (((row >> 1) & 1) << 2 | ((row >> 2) & 1) << 1 | ((row >> 3) & 1));
        if constexpr (UNITS == 16) return unit ^ ((row & 3) << 2 | ((row >> 2) & 3));
        const int moved = unit + ((row >> 2) & 3);
        return moved >= UNITS ? moved - UNITS : moved;
    }
    // Which unit of the row lies there.
    static __device__ __forceinline__ int unit_at(int row, int placed)
    {
        if constexpr (UNITS != 12) return place(row, placed);
        const int moved = placed - ((row >> 2) & 3);
        return moved < 0 ? moved + UNITS : moved;
    }
    __device__ __forceinline__ void put(int row, int unit, const AttnFrag<TERMS> &f) const
    {
#pragma unroll
        for (int t = 0; t < TERMS; ++t)
            *(pccnn_u32x4 *)(base + t * PLANE + row * DP + 8 * place(row, unit)) = __builtin_bit_cast(pccnn_u32x4, f.t[t]);
    }
    // Operand with the tile's rows as C's rows: the eight features of unit `unit` of row `row`.
    __device__ __forceinline__ AttnFrag<TERMS> rows(int row, int unit) const
    {
        AttnFrag<TERMS> f;
#pragma unroll
        for (int t = 0; t < TERMS; ++t)
            f.t[t] = __builtin_bit_cast(pccnn_bf16x8,
                                        *(const pccnn_u32x4 *)(base + t * PLANE + row * DP + 8 * place(row, unit)));
        return f;
    }
    // Operand with the tile's features as C's rows (feature col + (lane & 31)) and as k the sixteen tile rows from `row`,
    // in the order of C's registers: row + 4 half + {0..3}, row + 8 + 4 half + {0..3}.  The read exchanges a 4 x 16 block
    // among sixteen lanes: lane i brings four features of row i / 4 and gets feature i of all four rows.
    __device__ __forceinline__ AttnFrag<TERMS> columns(int row, int col, int lane) const
    {
        const int r = 4 * (lane >> 5) + ((lane & 15) >> 2), unit = (col + (lane & 16)) / 8 + ((lane & 3) >> 1);
        const int lo_at = r * DP + 8 * place(r, unit) + 4 * (lane & 1);
        const int hi_at = (r + 8) * DP + 8 * place(r + 8, unit) + 4 * (lane & 1);
        AttnFrag<TERMS> f;
#pragma unroll
        for (int t = 0; t < TERMS; ++t) {
            typedef __attribute__((address_space(3))) pccnn_i16x4 *lds_ptr;
            uint16_t *p = base + t * PLANE + row * DP;                // row: a multiple of 16, so place() sees r alone
            const pccnn_i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p + lo_at));
            const pccnn_i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p + hi_at));
            f.t[t] = __builtin_bit_cast(pccnn_bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        }
        return f;
    }
};

// A window on memory from `base` (the same in all lanes) for range-checked loads: an offset past 2^31 bytes reads zeros.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t attn_window(const void *base)
{
    return __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, 0x7fffffff, 0x00027000);
}
constexpr uint32_t kAttnNowhere = 0xfffffff0u;       // an offset past every window
// Memory to LDS without a register between: 16 bytes per lane, from its own offset in the window to `lds` + 16 * lane,
// `lds` the same in all lanes.  Lands by the next wait for vector memory (attn_landed).
__device__ __forceinline__ void attn_bring(__amdgpu_buffer_rsrc_t window, uint32_t offset, void *lds)
{
    typedef __attribute__((address_space(3))) void *lds_ptr;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(window, (lds_ptr)lds, 16, offset, 0, 0, 0);
}
// Everything this wavefront brought has landed; with the barrier behind it, everything the workgroup brought.
__device__ __forceinline__ void attn_landed()
{
    __builtin_amdgcn_s_waitcnt(0x0f70);              // vmcnt(0)
    __syncthreads();
}

// Operands are read from LDS a few products ahead of their use: a read takes as long as four products of 32 cycles, and the
// compiler, left alone, reads each one just before.  `load(i)` is the operand of the i-th of COUNT products, `use(i, f)` the
// product; the order of reads and products is kept, other instructions may move between them.
template <int TERMS> struct AttnAhead {
    static constexpr int DEPTH = TERMS == 3 ? 1 : 4;      // (three terms: six products to an operand)
    AttnFrag<TERMS> f[DEPTH];
    template <int COUNT, typename LOAD> __device__ __forceinline__ void prime(LOAD load)
    {
#pragma unroll
        for (int i = 0; i < DEPTH && i < COUNT; ++i) f[i] = load(i);
        __builtin_amdgcn_sched_barrier(0x6);              // VALU and SALU may cross
    }
    template <int COUNT, typename LOAD, typename USE> __device__ __forceinline__ void run(LOAD load, USE use)
    {
#pragma unroll
        for (int i = 0; i < COUNT; ++i) {
            const AttnFrag<TERMS> now = f[i % DEPTH];
            if (i + DEPTH < COUNT) f[i % DEPTH] = load(i + DEPTH);
            __builtin_amdgcn_sched_barrier(0x6);
            use(i, now);
            __builtin_amdgcn_sched_barrier(0x6);
        }
    }
};

// max(v, v of the lane 32 away)
__device__ __forceinline__ float attn_max_halves(float v)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
#endif
