// A cache of keys and values in 4 or 8 bits: its layout, and its elements as bfloat16 (included by .hip files only).
//
// Codes are (batch, kv_heads, keys, head_len) elements and scales (batch, kv_heads, keys, head_len / 32) bytes, for K and for V: a key head's
// rows follow one another, so that a workgroup which walks them reads whole cache lines (a row of 128 elements in 4 bits is half a line; with the
// heads of one key next to one another two workgroups, on different XCDs, would each fetch every line).
// Elements are e2m1 (4 bits, the lower half of a byte first) or e4m3 (8 bits); 32 of them share the scale 2^(byte - 127).  Either has 4 bits of
// precision at most and bfloat16 the range of 32 bits: every value is a bfloat16 exactly, made by one conversion for two of them.
// Byte 255 marks 32 elements with something that was not finite among them: all are NaN.
#pragma once

#include "fg_block.h"

namespace fg {
namespace cache {

using block::bf16x8;
using block::u32x4;

constexpr int kGroup = 32;                         // elements of one scale
template <int BITS> constexpr int kTopExponent = BITS == 4 ? 125 : 119;      // of a scale: with more, 6 (448) times it would be beyond 32 bits

// One of the two arrays of a cache, seen from a sequence's key head.
template <int D, int BITS> struct Rows {
    static constexpr int kBytes = D * BITS / 8, kScales = D / kGroup;
    const uint8_t *codes, *scales;
    __device__ __forceinline__ Rows(const void *c, const void *s, int64_t head, int64_t keys)
        : codes(static_cast<const uint8_t *>(c) + head * keys * kBytes), scales(static_cast<const uint8_t *>(s) + head * keys * kScales) {}
    __device__ __forceinline__ Rows(const Rows &r, int64_t key) : codes(r.codes + key * kBytes), scales(r.scales + key * kScales) {}     // from a key on
};

__device__ __forceinline__ float scale_of(unsigned byte) { return __uint_as_float(byte << 23); }     // as the conversions read it: its exponent alone

// Eight elements: the one (4 bits) or two (8 bits) words that hold them, times the scale, as bfloat16 (numbers below 2^-126 less exactly) or in 32 bits.
template <int BITS, typename T = __bf16> __device__ __forceinline__ block::V8<T> values(const uint32_t *word, float scale) {
    typedef T T2 __attribute__((ext_vector_type(2)));
    T2 a, b, c, d;
    if constexpr (BITS == 4 && sizeof(T) == 2) {
        a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word[0], scale, 0);
        b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word[0], scale, 1);
        c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word[0], scale, 2);
        d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word[0], scale, 3);
    } else if constexpr (BITS == 4) {
        a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word[0], scale, 0);
        b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word[0], scale, 1);
        c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word[0], scale, 2);
        d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word[0], scale, 3);
    } else if constexpr (sizeof(T) == 2) {
        a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word[0], scale, false);
        b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word[0], scale, true);
        c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word[1], scale, false);
        d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word[1], scale, true);
    } else {
        a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(word[0], scale, false);
        b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(word[0], scale, true);
        c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(word[1], scale, false);
        d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(word[1], scale, true);
    }
    return block::V8<T>{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// A number as it is rounded to T: an element may be larger than the value it came from (65504 is held as 65536), and float16 takes no such number.
template <typename T> __device__ __forceinline__ float within(float f) {
    if constexpr (std::is_same<T, _Float16>::value) return f != f ? f : fminf(fmaxf(f, -65504.f), 65504.f);
    else return f;
}

// FG_OK, or why the arrays cannot be such a cache.
int check(const fg_kv_cache *c);

}  // namespace cache
}  // namespace fg
