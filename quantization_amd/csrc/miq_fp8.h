// Device-side building blocks of the block-scaled 8-bit floating point operators: e4m3 codes, block maxima, and the
// scale of a block.
//
// A block is 128 consecutive columns (of one row for activations, of 128 rows for weights).  With a the largest finite
// magnitude in the block, taken as at least 448 * 2^-126:
//     scale = a / 448                 (fp32, IEEE division; a normal number, never 0)
//     code  = e4m3(x * (448 / a))     (fp32 quotient, once per block; fp32 product; round-half-even to OCP e4m3)
// so that |x * (448 / a)| <= 448 * (1 + 2^-22): the conversion never overflows (e4m3 rounds everything below 464 to 448).
// An element that is not finite becomes the NaN code (e4m3 has no infinity) and does not enter its block's maximum, so it
// does not spoil its neighbours.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "miq_common.h"

namespace miq {

constexpr int kBlockK = 128;                                  // columns that share a scale
constexpr float kTopE4m3 = 448.0f;
constexpr float kLeastMax = 448.0f * 1.17549435e-38f;         // 448 * 2^-126
constexpr uint32_t kInfBits = 0x7f800000u;

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

// Four floats as four packed e4m3 codes (v_cvt_pk_fp8_f32: round-half-even, NaN -> NaN code).
__device__ __forceinline__ uint32_t pack4_e4m3(float a, float b, float c, float d) {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true));
}

// Magnitudes compare as their bit patterns; everything at or above kInfBits is an infinity or a NaN.
__device__ __forceinline__ uint32_t magnitude_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// A value that is not finite takes no part in its block's maximum ...
__device__ __forceinline__ uint32_t finite_magnitude_bits(float x) {
    const uint32_t b = magnitude_bits(x);
    return b < kInfBits ? b : 0u;
}
// ... and becomes the NaN code.
__device__ __forceinline__ float infinite_to_nan(float x) {
    return magnitude_bits(x) < kInfBits ? x : __uint_as_float(0x7fc00000u);
}

// Unsigned maximum over the 16 lanes of a DPP row, in all of them.
template <int CTRL>
__device__ __forceinline__ uint32_t max_dpp(uint32_t v) {
    const uint32_t o = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xf, 0xf, false));
    return o > v ? o : v;
}
__device__ __forceinline__ uint32_t max_over_16_lanes(uint32_t v) {
    v = max_dpp<0x128>(v);   // row_ror:8
    v = max_dpp<0x124>(v);
    v = max_dpp<0x122>(v);
    return max_dpp<0x121>(v);
}

struct BlockScale {
    float scale, inv;   // a / 448 and 448 / a
};
__device__ __forceinline__ BlockScale block_scale(uint32_t max_bits) {
    const float a = fmaxf(__uint_as_float(max_bits), kLeastMax);
    return {__fdiv_rn(a, kTopE4m3), __fdiv_rn(kTopE4m3, a)};
}

// A vector at any address: the hardware takes it, so a row that starts anywhere is read and written like an aligned one but for
// its last elements (2048x14335 bf16 codes 19.7 us, element by element 57; aligned, 14336, 16.5).  Aligned rows pass the caches
// by; of the others neighbouring lanes and waves share lines, which the caches then join (19.7 us; passing them by 24.5).
typedef u32x4 u32x4_any __attribute__((aligned(1)));
typedef u32x2 u32x2_any __attribute__((aligned(1)));
template <bool NT>
__device__ __forceinline__ u32x4 load16(const void* p) {
    if constexpr (NT) return __builtin_nontemporal_load(static_cast<const u32x4_any*>(p));
    else return *static_cast<const u32x4_any*>(p);
}

// Eight consecutive elements of floating storage type DT as floats.  `n` of them are inside the row (the others read as
// 0); VEC: n is 0 or 8 and the address a multiple of 16 bytes; NT: read once, kept out of the caches.
template <int DT, bool VEC, bool NT = true>
__device__ __forceinline__ void load8(const void* base, int64_t index, int n, float (&f)[8]) {
    if constexpr (DT == MIQ_F32) {
        const float* p = static_cast<const float*>(base) + index;
        u32x4 a = {0, 0, 0, 0}, b = {0, 0, 0, 0};
        if (n == 8) {
            a = load16<NT && VEC>(p);
            b = load16<NT && VEC>(p + 4);
        } else if (!VEC) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (i < n) a[i] = __float_as_uint(p[i]);
                if (4 + i < n) b[i] = __float_as_uint(p[4 + i]);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[i] = __uint_as_float(a[i]);
            f[4 + i] = __uint_as_float(b[i]);
        }
    } else {
        const uint16_t* p = static_cast<const uint16_t*>(base) + index;
        u32x4 v = {0, 0, 0, 0};
        if (n == 8) {
            v = load16<NT && VEC>(p);
        } else if (!VEC) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < n) v[i >> 1] |= static_cast<uint32_t>(p[i]) << (16 * (i & 1));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (DT == MIQ_BF16) {
                f[2 * i] = __uint_as_float(v[i] << 16);
                f[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
            } else {
                typedef _Float16 h2 __attribute__((ext_vector_type(2)));
                const h2 h = __builtin_bit_cast(h2, static_cast<uint32_t>(v[i]));
                f[2 * i] = static_cast<float>(h[0]);
                f[2 * i + 1] = static_cast<float>(h[1]);
            }
        }
    }
}

// Eight codes at q[index ...], `n` of them inside the row.
template <bool VEC>
__device__ __forceinline__ void store8_codes(uint8_t* q, int64_t index, int n, const uint32_t (&c)[2]) {
    if (n == 8) {
        const u32x2 v = {c[0], c[1]};
        if constexpr (VEC) __builtin_nontemporal_store(v, reinterpret_cast<u32x2*>(q + index));
        else *reinterpret_cast<u32x2_any*>(q + index) = v;
    } else if (!VEC) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) q[index + i] = static_cast<uint8_t>(c[i >> 2] >> (8 * (i & 3)));
    }
}

// The codes of eight values of a block whose largest finite magnitude is max_bits; `spoiled`: some value of the wave is
// not finite.
__device__ __forceinline__ void codes8(float (&f)[8], float inv, bool spoiled, uint32_t (&c)[2]) {
    if (spoiled) {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = infinite_to_nan(f[i]);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
        c[h] = pack4_e4m3(__fmul_rn(f[4 * h], inv), __fmul_rn(f[4 * h + 1], inv), __fmul_rn(f[4 * h + 2], inv),
                          __fmul_rn(f[4 * h + 3], inv));
}

// Scale and codes of eight of a block's 128 values, the other lanes of this lane's row of 16 holding the rest.
__device__ __forceinline__ float quantize8_in_row(float (&f)[8], uint32_t (&c)[2]) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t b = magnitude_bits(f[i]);
        top = b > top ? b : top;
    }
    top = max_over_16_lanes(top);
    const bool spoiled = __any(top >= kInfBits);   // rare: the whole wave takes the careful way
    if (spoiled) {
        top = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t b = finite_magnitude_bits(f[i]);
            top = b > top ? b : top;
        }
        top = max_over_16_lanes(top);
    }
    const BlockScale s = block_scale(top);
    codes8(f, s.inv, spoiled, c);
    return s.scale;
}

}  // namespace miq
