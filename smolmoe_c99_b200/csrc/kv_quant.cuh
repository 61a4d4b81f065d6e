// The 8-bit key/value cache: what a page holds and how a value is taken from it.
//
// A row (the head_dim values of one position and kv head) is held as one byte a value and one byte a row: the exponent of
// a power-of-two scale, plus 127. Largest code: 448 = 1.75 * 2^8 (e4m3), 127 = 1.984375 * 2^6 (int8). With amax = m * 2^E
// the largest magnitude of the row (1 <= m < 2), the exponent is
//   e = E - 8 + [m > 1.75]  or  E - 6 + [m > 1.984375], at least kLeastExponent,
// the smallest for which no code overflows; code = round to nearest even of x * 2^-e, value = code * 2^e.
// Why a power of two: e4m3 is a floating-point format, so a finer scale would give it nothing (int8, whose steps are even, loses
// up to a bit against a scale that takes the row's largest value to 127); x * 2^-e and code * 2^e are exact; and a code of at most 7 significant bits times a power of two is a bfloat16 number, so a kernel that reads the
// cache as bfloat16 and one that multiplies codes see the same values.
// A row with an infinity or a NaN has no scale: its byte is kNoScale, its codes are 0, and it reads back as NaN whole (the
// byte's bits as a float are infinity, times 0). Codes that were written are therefore always finite. (A value that rounds up to
// 2^128, from 1.9375 * 2^127 in e4m3 and 1.984375 * 2^127 in int8, has no float and reads back as infinity.)
//
// Pools, per layer: codes [pages, kv_heads, kPageSize, head_dim], exponents [pages, kv_heads, kPageSize] (one each for
// keys and values); position p of a sequence lies on page page_table[slot][p / kPageSize]. Every position is kept.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

namespace sm {

enum QuantFormat : int { QUANT_FP8 = 0, QUANT_INT8 = 1 };

constexpr int kLeastExponent = -100;   // rows whose largest value is below about 2^-92 lose bits (and are zero below 2^-110)
constexpr int kNoScale = 255;

// Codes in the library's error word for a slot, position or page that lies outside the page table or the pools: the access
// is left out (rows are not written, or read as zeros). Reading back also reports a sequence that is longer than the pages it reads,
// attention lengths that are not those of the host.
constexpr int kBadPlaceInStore = 31, kBadPlaceInLoad = 32, kBadPlaceInAttention = 33;

// The page of a sequence's positions 64 * index .. 64 * index + 63, or -1 where there is none.
struct QuantPages {
    const int32_t* table;        // [slots][stride]
    int slots, stride;
    long long pages;             // of the pools

    __device__ __forceinline__ int at(int slot, int index) const {
        if ((unsigned)slot >= (unsigned)slots || (unsigned)index >= (unsigned)stride) return -1;
        const int page = table[(size_t)slot * stride + index];
        return page >= 0 && page < pages ? page : -1;
    }
};

// What kv_quant_load reads back of a sequence for a kernel that attends over it: `count` pages from `first` on, those that a token
// of the step sees in `window` (0: all) and the neighbour that shares 128 positions with the first of them; at most page most - 1.
struct PagesRead {
    int first, count;
};
__device__ __forceinline__ PagesRead pages_read(int start, int end, int window, int most) {
    const int first = (window > 0 ? max(0, start - window + 1) : 0) / 128 * (128 / kPageSize);
    return {first, max(min((end + kPageSize - 1) / kPageSize, most) - first, 0)};
}

// 2^e for -126 <= e <= 127
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }
// the factor of a row from its byte (infinity for kNoScale: its codes are 0, so the product is NaN; 0 for a row never written)
__device__ __forceinline__ float scale_of(int byte) { return __int_as_float(byte << 23); }

// A row's byte from the bits of its largest magnitude (which order as the magnitudes do; NaN and infinity are the largest).
template <int FMT>
__device__ __forceinline__ int scale_byte(uint32_t amax_bits) {
    if (amax_bits >= 0x7f800000u) return kNoScale;
    const int E = (int)(amax_bits >> 23) - 127;
    const uint32_t m = amax_bits & 0x7fffffu;
    const int e = FMT == QUANT_FP8 ? E - 8 + (m > 0x600000u ? 1 : 0) : E - 6 + (m > 0x7e0000u ? 1 : 0);
    return max(e, kLeastExponent) + 127;
}

// Four scaled values as four codes (lowest byte first), rounded to nearest even.
template <int FMT>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
    if (FMT == QUANT_FP8) {
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
        return lo | (hi << 16);
    }
    return (uint32_t)(__float2int_rn(a) & 255) | ((uint32_t)(__float2int_rn(b) & 255) << 8) |
           ((uint32_t)(__float2int_rn(c) & 255) << 16) | ((uint32_t)(__float2int_rn(d) & 255) << 24);
}

// Four codes (lowest byte first) as two pairs of half-precision numbers (exact in both formats). int8: a code plus 128 put into the last bits of
// 1,024.0 gives 1,152 + code; the subtraction is exact.
template <int FMT>
__device__ __forceinline__ void decode4(uint32_t codes, uint32_t& lo, uint32_t& hi) {
    if (FMT == QUANT_FP8) {
        asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
            : "=r"(lo), "=r"(hi) : "r"(codes));
    } else {
        const uint32_t u = codes ^ 0x80808080u;
        const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
        const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
        const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), bias);
        const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&b), bias);
        lo = *reinterpret_cast<const uint32_t*>(&x);
        hi = *reinterpret_cast<const uint32_t*>(&y);
    }
}
template <int FMT>
__device__ __forceinline__ void decode4(uint32_t codes, float (&v)[4]) {
    uint32_t lo, hi;
    decode4<FMT>(codes, lo, hi);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo)), b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
}

}  // namespace sm
