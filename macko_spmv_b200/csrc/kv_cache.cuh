// The paged key/value cache in 8 bits: what its kernels share. Host side: the checks of the two argument structs.
// Device side: which rows belong to which sequence, where a token lies, and codes to and from floating point.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace macko {

// macko_kv_cache for the kernels. A page of one head is page_size x head_dim consecutive bytes.
struct CacheView {
    uint8_t *k, *v;
    float *k_scale, *v_scale;
    long long k_stride, v_stride;              // bytes between pages
    long long k_scale_stride, v_scale_stride;  // floats between pages
    int pages, kv_heads, page_log2, head_dim;
};

// macko_kv_rows for the kernels.
struct RowsView {
    const int *table, *lengths, *start;   // start: null where every sequence has one row
    long long table_stride;
    int width, capacity;                  // pages and tokens that a sequence can have
    int sequences, rows;
};

// Status of the structs; fills the views.
int check_cache(const char *what, const macko_kv_cache *cache, CacheView *view);
int check_rows(const char *what, const macko_kv_rows *rows, int page_size, RowsView *view);

// Scales are powers of two from 2^-64 on; smaller ones (a user's own) are read as 2^-64, so that a page without any weight still
// has its share of the softmax sum.
constexpr float kLowestScale = 5.421010862427522e-20f;

#ifdef __CUDACC__

// Rows [first, first + count) of the call are the last `count` of the sequence's `length` tokens. Whatever the device arrays
// hold, the rows are rows of the call and the length is not negative; positions may still lie outside 0 .. capacity - 1. (The arrays
// may have been written by the kernel in front, under which this one may have begun: they are read past the L1 cache.)
struct Sequence {
    int first, count, length;
    __device__ __forceinline__ int begin() const { return length - count; }   // position of the first row
};

__device__ __forceinline__ Sequence sequence_at(const RowsView &r, int i)
{
    Sequence s;
    s.length = max(__ldcg(r.lengths + i), 0);
    if (r.start == nullptr) {
        s.first = i;
        s.count = 1;
    } else {
        s.first = min(max(__ldcg(r.start + i), 0), r.rows);
        s.count = min(max(__ldcg(r.start + i + 1), s.first), r.rows) - s.first;
    }
    return s;
}

// Page of the cache that holds a position below the capacity, or -1 where the table's entry is no page.
__device__ __forceinline__ int page_at(const CacheView &c, const RowsView &r, int sequence, int position)
{
    const int page = __ldcg(r.table + (long long)sequence * r.table_stride + (position >> c.page_log2));
    return (unsigned)page < (unsigned)c.pages ? page : -1;
}

// a * b - c * d rounded to odd in fp32: the exact value where it fits, else the neighbour whose last bit is set. Rounding that to
// 22 bits or fewer gives what rounding the exact value gives, ties included. Exact for factors of up to 12 bits (fp16, bf16).
__device__ __forceinline__ float difference_to_odd(float a, float b, float c, float d)
{
    const float p = -c * d;
    const float down = __fmaf_rd(a, b, p), up = __fmaf_ru(a, b, p);
    return (__float_as_uint(down) & 1u) ? down : up;
}

template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t raw)
{
    if (BF16) return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&raw));
    return __half22float2(*reinterpret_cast<const __half2 *>(&raw));
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi)
{
    uint32_t raw;
    if (BF16) *reinterpret_cast<__nv_bfloat162 *>(&raw) = __floats2bfloat162_rn(lo, hi);
    else *reinterpret_cast<__half2 *>(&raw) = __floats2half2_rn(lo, hi);
    return raw;
}

// 16 bytes of global memory, or zeros; without a branch, so that many of these are under way at a time.
__device__ __forceinline__ void load_if(uint4 &x, const void *p, bool there)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\tmov.b32 %2, 0;\n\tmov.b32 %3, 0;\n\t"
                 "@p ld.global.cg.v4.b32 {%0, %1, %2, %3}, [%4];\n\t}"
                 : "=&r"(x.x), "=&r"(x.y), "=&r"(x.z), "=&r"(x.w) : "l"(p), "r"((int)there));
}

// The scale of a page's values as the softmax counts it: NaN stays NaN.
__device__ __forceinline__ float value_scale(float scale) { return scale < kLowestScale ? kLowestScale : scale; }

// 1 / scale; the quick division by more than 2^126 would be zero.
__device__ __forceinline__ float inverse_scale(float scale) { return __fdividef(0.25f, 0.25f * scale); }

// Four codes, as they lie in memory, as two pairs of fp16 values, exactly. int8: the byte with its sign bit flipped, put under
// the exponent of 1024, is 1024 + 128 + code; 1152 is taken off again.
template <bool E4M3>
__device__ __forceinline__ void codes_to_half(uint32_t codes, uint32_t &lo, uint32_t &hi)
{
    if (E4M3) {
        asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(lo), "=r"(hi) : "r"(codes));
    } else {
        const uint32_t x = codes ^ 0x80808080u;
        const __half2 off = __half2half2(__ushort_as_half((unsigned short)0x6480));   // 1152
        const uint32_t a = __byte_perm(x, 0x64646464u, 0x4140), b = __byte_perm(x, 0x64646464u, 0x4342);
        const __half2 l = __hsub2(*reinterpret_cast<const __half2 *>(&a), off), h = __hsub2(*reinterpret_cast<const __half2 *>(&b), off);
        lo = *reinterpret_cast<const uint32_t *>(&l);
        hi = *reinterpret_cast<const uint32_t *>(&h);
    }
}

// Four values, already divided by their scale, as codes: to nearest even, at most the largest code.
template <bool E4M3>
__device__ __forceinline__ uint32_t codes_from_float(float a, float b, float c, float d)
{
    if (E4M3) {
        uint16_t lo, hi;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
        return (uint32_t)lo | (uint32_t)hi << 16;
    }
    const auto code = [](float x) { return (uint32_t)__float2int_rn(fminf(fmaxf(x, -127.f), 127.f)) & 0xffu; };
    return code(a) | code(b) << 8 | code(c) << 16 | code(d) << 24;
}

#endif  // __CUDACC__

}  // namespace macko
