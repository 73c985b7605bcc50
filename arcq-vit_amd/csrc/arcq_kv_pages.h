// The pages of a key/value cache (arcq_kv_pages of include/arcq_hip.h): host checks and the 16-bit types of what passes
// through them.
#pragma once

#include "arcq_common.h"

namespace arcq {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float float4_t __attribute__((ext_vector_type(4)));
typedef float float16_t __attribute__((ext_vector_type(16)));

// Two floats rounded to nearest even into one register.
__device__ __forceinline__ uint32_t pack2(float a, float b, _Float16)
{
    const half2_t v = {static_cast<_Float16>(a), static_cast<_Float16>(b)};
    return __builtin_bit_cast(uint32_t, v);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __bf16)
{
    const bf16x2_t v = {static_cast<__bf16>(a), static_cast<__bf16>(b)};
    return __builtin_bit_cast(uint32_t, v);
}
// The two values of a register as floats.
__device__ __forceinline__ void unpack2(uint32_t w, float &a, float &b, _Float16)
{
    const half2_t v = __builtin_bit_cast(half2_t, w);
    a = static_cast<float>(v[0]);
    b = static_cast<float>(v[1]);
}
__device__ __forceinline__ void unpack2(uint32_t w, float &a, float &b, __bf16)
{
    a = __builtin_bit_cast(float, w << 16);
    b = __builtin_bit_cast(float, w & 0xffff0000u);
}

// Exponents that FP8 rows of a type may have: the largest keeps every value of the row finite in the type (448 * 2^7 is the
// last below 65 504, 448 * 2^119 the last below 2^128); the smallest loses nothing that the type can hold (fp16: 2^-14 times
// the FP8 subnormals' step of 2^-9 is 2^-23) or keeps every value a normal number (bf16).
template <typename T> struct ExponentRange;
template <> struct ExponentRange<_Float16> { static constexpr int lo = -14, hi = 7; };
template <> struct ExponentRange<__bf16> { static constexpr int lo = -110, hi = 119; };

// Null, or what is wrong with the pages.
inline int check_pages(const char *fn, const arcq_kv_pages &p, int dtype)
{
    if (dtype != ARCQ_F16 && dtype != ARCQ_BF16) return fail(ARCQ_ERR_DTYPE, "%s: dtype must be ARCQ_F16 or ARCQ_BF16", fn);
    if (p.dtype != ARCQ_FP8 && p.dtype != dtype)
        return fail(ARCQ_ERR_DTYPE, "%s: 16-bit pages and the rows must have one dtype", fn);
    if (p.num_pages < 0 || p.heads < 0 || p.page_size < 16 || (p.page_size & (p.page_size - 1)) != 0 || p.page_size > (1 << 20))
        return fail(ARCQ_ERR_SHAPE, "%s: page_size must be a power of two, 16 to 2^20 (got %lld)", fn, static_cast<long long>(p.page_size));
    if (p.head_dim < 16 || p.head_dim > 256 || p.head_dim % 16 != 0)
        return fail(ARCQ_ERR_UNSUPPORTED, "%s: head_dim must be a multiple of 16, at most 256 (got %lld)", fn, static_cast<long long>(p.head_dim));
    if (p.num_pages >= (int64_t(1) << 31) || p.heads > 65535) return fail(ARCQ_ERR_SHAPE, "%s: too many pages or heads", fn);
    return ARCQ_OK;
}
// The pointers, once there is something to do.
inline int check_page_pointers(const char *fn, const arcq_kv_pages &p)
{
    if (p.num_pages == 0) return ARCQ_OK;
    if (!p.k || !p.v || (p.dtype == ARCQ_FP8 && (!p.k_exponents || !p.v_exponents))) return fail(ARCQ_ERR_NULL, "%s: NULL pages", fn);
    if (!aligned(p.k, 16) || !aligned(p.v, 16) || !aligned(p.k_exponents, 16) || !aligned(p.v_exponents, 16))
        return fail(ARCQ_ERR_ALIGN, "%s: pages must be 16-byte aligned", fn);
    return ARCQ_OK;
}
// Do all rows [rows, heads] of 16-bit values lie on 16-byte boundaries?  (A dimension of one entry has any stride.)
inline bool rows_aligned(const void *p, int64_t rows, int64_t row_stride, int64_t heads, int64_t head_stride)
{
    return aligned(p, 16) && (rows <= 1 || row_stride % 8 == 0) && (heads <= 1 || head_stride % 8 == 0);
}
inline int log2_of(int64_t power)
{
    int n = 0;
    while ((int64_t(1) << n) < power) ++n;
    return n;
}

}  // namespace arcq
