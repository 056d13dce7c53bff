// Element types of the feature operators (layer norm, rotary positions, attention): f32, or bf16 as bit patterns.
// Values are f32 in registers; a bf16 result is rounded when it is stored, to nearest even (what attention's products round
// before is said there).
#pragma once
#include "common.h"

static inline int pccnn_type_ok(int type) { return type == PCCNN_TYPE_F32 || type == PCCNN_TYPE_BF16; }
static inline int pccnn_type_bytes(int type) { return type == PCCNN_TYPE_BF16 ? 2 : 4; }
// Whether rows `stride` elements apart, from `p` on, all start at a multiple of `bytes`.
static inline bool pccnn_rows_aligned(const void *p, int64_t stride, int type, int bytes)
{
    return (uintptr_t)p % (uintptr_t)bytes == 0 && (stride * pccnn_type_bytes(type)) % bytes == 0;
}

#ifdef __HIPCC__
typedef __bf16 pccnn_bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 pccnn_bf16x8 __attribute__((ext_vector_type(8)));
typedef float pccnn_f32x2 __attribute__((ext_vector_type(2)));
typedef float pccnn_f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned int pccnn_u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int pccnn_u32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float pccnn_bf16_value(uint16_t bits) { return __uint_as_float((uint32_t)bits << 16); }

// Two values rounded to bf16 (nearest even), the first in the low half.
__device__ __forceinline__ uint32_t pccnn_bf16_pair(float a, float b)
{
    const pccnn_f32x2 v = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, pccnn_bf16x2));
}

// COUNT consecutive elements to and from f32.  The address is a multiple of min(16, COUNT * sizeof(T)) bytes.
template <int COUNT> __device__ __forceinline__ void pccnn_load(const float *p, float (&v)[COUNT])
{
    if constexpr (COUNT % 4 == 0) {
#pragma unroll
        for (int i = 0; i < COUNT; i += 4) {
            const float4 q = *(const float4 *)(p + i);
            v[i] = q.x; v[i + 1] = q.y; v[i + 2] = q.z; v[i + 3] = q.w;
        }
    } else if constexpr (COUNT == 2) {
        const float2 q = *(const float2 *)p;
        v[0] = q.x; v[1] = q.y;
    } else {
        static_assert(COUNT == 1, "1, 2 or a multiple of 4");
        v[0] = *p;
    }
}
template <int COUNT> __device__ __forceinline__ void pccnn_load(const uint16_t *p, float (&v)[COUNT])
{
    if constexpr (COUNT == 1) {
        v[0] = pccnn_bf16_value(*p);
    } else {
        uint32_t w[COUNT / 2];
        if constexpr (COUNT % 8 == 0) {
#pragma unroll
            for (int i = 0; i < COUNT / 8; ++i) {
                const uint4 q = *(const uint4 *)(p + 8 * i);
                w[4 * i] = q.x; w[4 * i + 1] = q.y; w[4 * i + 2] = q.z; w[4 * i + 3] = q.w;
            }
        } else if constexpr (COUNT == 4) {
            const uint2 q = *(const uint2 *)p;
            w[0] = q.x; w[1] = q.y;
        } else {
            static_assert(COUNT == 2, "1, 2, 4 or a multiple of 8");
            w[0] = *(const uint32_t *)p;
        }
#pragma unroll
        for (int i = 0; i < COUNT / 2; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
}
template <int COUNT> __device__ __forceinline__ void pccnn_store(float *p, const float (&v)[COUNT])
{
    if constexpr (COUNT % 4 == 0) {
#pragma unroll
        for (int i = 0; i < COUNT; i += 4) *(float4 *)(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
    } else if constexpr (COUNT == 2) {
        *(float2 *)p = make_float2(v[0], v[1]);
    } else {
        *p = v[0];
    }
}
template <int COUNT> __device__ __forceinline__ void pccnn_store(uint16_t *p, const float (&v)[COUNT])
{
    if constexpr (COUNT == 1) {
        *p = (uint16_t)pccnn_bf16_pair(v[0], v[0]);
    } else {
        uint32_t w[COUNT / 2];
#pragma unroll
        for (int i = 0; i < COUNT / 2; ++i) w[i] = pccnn_bf16_pair(v[2 * i], v[2 * i + 1]);
        if constexpr (COUNT % 8 == 0) {
#pragma unroll
            for (int i = 0; i < COUNT / 8; ++i)
                *(uint4 *)(p + 8 * i) = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
        } else if constexpr (COUNT == 4) {
            *(uint2 *)p = make_uint2(w[0], w[1]);
        } else {
            *(uint32_t *)p = w[0];
        }
    }
}
// One element of a tensor whose type is known at run time (weights: a few values per thread).
__device__ __forceinline__ float pccnn_element(const void *p, int type, int64_t i)
{
    return type == PCCNN_TYPE_BF16 ? pccnn_bf16_value(((const uint16_t *)p)[i]) : ((const float *)p)[i];
}
__device__ __forceinline__ void pccnn_set_element(void *p, int type, int64_t i, float v)
{
    if (type == PCCNN_TYPE_BF16)
        ((uint16_t *)p)[i] = (uint16_t)pccnn_bf16_pair(v, v);
    else
        ((float *)p)[i] = v;
}
#endif
