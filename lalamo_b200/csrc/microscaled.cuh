// Microscaled rows (the OCP microscaling formats): elements of 8 bits (e4m3) or 4 (e2m1) with a power of two as the scale of every 32 columns of
// a row.  Layout, `padded` being the width made up to whole 128s:
//     codes  [rows, padded * bits / 8] bytes; of 4-bit elements the even column is the lower half of its byte; columns past the width hold zeros
//     scales [ceil(rows / 128), padded / 128, 512] bytes b, each 2^(b - 127), 255 not a number: that of row r and columns 32 c ... 32 c + 31 is byte
//            (r % 32) * 16 + (r % 128) / 32 * 4 + c % 4 of tile [r / 128, c / 4]
// A tile of scales is what tcgen05.cp sets down in four columns of tensor memory for 128 rows and 128 columns, so that a product copies scales as it
// copies elements.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

namespace lb {

constexpr int kScaleTileBytes = 512;
constexpr int kNoNumber = 255;   // the scale of a block that holds a NaN or an infinity: every value of it is NaN

// Where the scales of row `row` and columns 128 * chunk ... + 127 lie: four consecutive bytes, aligned.
__device__ __forceinline__ size_t scale_word(int row, int chunk, int chunks) {
    return (static_cast<size_t>(row >> 7) * chunks + chunk) * kScaleTileBytes + (row & 31) * 16 + ((row >> 5) & 3) * 4;
}

// The scale of a block whose largest magnitude has these float32 bits: 2^(floor(log2 largest) - emax), emax the exponent of the format's largest
// element (8 of 448, 2 of 6).  With biased exponents that is a subtraction, and what falls below 2^-127 (zeros and subnormals among it) takes that.
template <int BITS>
__device__ __forceinline__ int scale_byte(uint32_t largest_bits) {
    const int exponent = static_cast<int>(largest_bits >> 23);
    return exponent == 255 ? kNoNumber : max(exponent - (BITS == 8 ? 8 : 2), 0);
}

// One over a scale, exact: the byte of a number is at most 254 - 2 (and what 255 gives is not looked at).
__device__ __forceinline__ float scale_inverse(int byte) { return __uint_as_float(static_cast<uint32_t>(254 - byte) << 23); }

// A scale as float32: 2^-127 is a subnormal.
__device__ __forceinline__ float scale_value(int byte) {
    return byte == kNoNumber ? __uint_as_float(0x7fffffffu) : byte == 0 ? __uint_as_float(0x00400000u) : __uint_as_float(static_cast<uint32_t>(byte) << 23);
}

// Four elements as e4m3 bytes, the first lowest; to the nearest, ties to even, what is larger than 448 becomes that.
__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d) {
    uint16_t low, high;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(low) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(high) : "f"(d), "f"(c));
    return static_cast<uint32_t>(low) | (static_cast<uint32_t>(high) << 16);
}
// Eight elements as e2m1 halves of bytes, the first lowest; likewise, with 6.
__device__ __forceinline__ uint32_t pack_e2m1(const float (&v)[8]) {
    uint32_t packed;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(packed)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return packed;
}

// The elements of eight consecutive columns, without their scale.
template <int BITS>
__device__ __forceinline__ void unpack_eight(uint2 codes, float (&v)[8]) {
    uint32_t pairs[4];   // float16, which holds every element of both formats
    if constexpr (BITS == 8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint16_t two = static_cast<uint16_t>((i < 2 ? codes.x : codes.y) >> (16 * (i & 1)));
            asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(pairs[i]) : "h"(two));
        }
    } else {
        asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
            "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
            "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
            "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
            "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
            "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
            : "=r"(pairs[0]), "=r"(pairs[1]), "=r"(pairs[2]), "=r"(pairs[3])
            : "r"(codes.x));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 both = __half22float2(*reinterpret_cast<const __half2*>(&pairs[i]));
        v[2 * i] = both.x;
        v[2 * i + 1] = both.y;
    }
}

// The larger of two magnitudes; a NaN is above all numbers (and stays one with an exponent of all ones).
__device__ __forceinline__ float larger_size(float a, float b) {
    float c;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(fabsf(a)), "f"(fabsf(b)));
    return c;
}

// The smaller and the larger of two numbers, a NaN if either is one (fminf and fmaxf give the other).
__device__ __forceinline__ float at_most(float a, float limit) {
    float c;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(limit));
    return c;
}
__device__ __forceinline__ float at_least(float a, float limit) {
    float c;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(limit));
    return c;
}

// Quantises eight or sixteen consecutive columns a lane: four (two) lanes hold a block, sixteen (eight) the 128 columns under one word of scales.  All lanes of
// the warp take part.  Returns that word (the same in all of them); `codes` has four bytes, or two bytes of halves, for every four columns.  (What the
// elements of a block are that has no number for a scale says nothing.)
template <int BITS, int COUNT>
__device__ __forceinline__ uint32_t quantise(const float (&v)[COUNT], uint32_t (&codes)[COUNT * BITS / 32]) {
    constexpr int kLanes = 32 / COUNT;   // of a block
    float largest = larger_size(v[0], v[1]);
#pragma unroll
    for (int i = 2; i < COUNT; i += 2) largest = larger_size(largest, larger_size(v[i], v[i + 1]));
#pragma unroll
    for (int offset = 1; offset < kLanes; offset <<= 1) largest = larger_size(largest, __shfl_xor_sync(0xffffffffu, largest, offset));
    const int byte = scale_byte<BITS>(__float_as_uint(largest) & 0x7fffffffu);
    const float inverse = scale_inverse(byte);
    if constexpr (BITS == 8) {
#pragma unroll
        for (int i = 0; i < COUNT / 4; ++i) codes[i] = pack_e4m3(v[4 * i] * inverse, v[4 * i + 1] * inverse, v[4 * i + 2] * inverse, v[4 * i + 3] * inverse);
    } else {
#pragma unroll
        for (int i = 0; i < COUNT / 8; ++i) {
            float scaled[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) scaled[e] = v[8 * i + e] * inverse;
            codes[i] = pack_e2m1(scaled);
        }
    }
    uint32_t word = static_cast<uint32_t>(byte) << ((threadIdx.x / kLanes & 3) * 8);
    word |= __shfl_xor_sync(0xffffffffu, word, kLanes);
    word |= __shfl_xor_sync(0xffffffffu, word, 2 * kLanes);
    return word;
}

// Its codes, at a place that their bytes divide.
template <int WORDS>
__device__ __forceinline__ void store_codes(unsigned char* to, const uint32_t (&codes)[WORDS]) {
    if constexpr (WORDS == 4) *reinterpret_cast<uint4*>(to) = make_uint4(codes[0], codes[1], codes[2], codes[3]);
    else if constexpr (WORDS == 2) *reinterpret_cast<uint2*>(to) = make_uint2(codes[0], codes[1]);
    else *reinterpret_cast<uint32_t*>(to) = codes[0];
}

// g Phi(g).  A block has a scale of its own, and one of far negative gates would show the last bits of 1 + erf as its values: for those g Phi(g) = -q and else g - q, with
// q = |g| erfc(z) / 2, z = |g| / sqrt 2.  exp(z^2) erfc(z) is t P(t) with t = 1 / (1 + 0.6 z) and a polynomial of degree 7, fitted for the smallest relative error (3.1e-7 for
// z up to 10); halves are in its coefficients.  (4,096 tokens, 6912 x 1536, sustained: 98 us, 87 to 96 with erff and 118 with erfcf; 777 tokens 21.1, 20.9 and 25.9.)
__device__ __forceinline__ float gelu(float g) {
    const float size = fabsf(g), t = __fdividef(1.0f, 1.0f + 0.42426407f * size);
    float p = -0.04604113f;
    p = p * t + 0.2059727f;
    p = p * t - 0.32222763f;
    p = p * t + 0.1418851f;
    p = p * t + 0.036705531f;
    p = p * t + 0.1458007f;
    p = p * t + 0.16862454f;
    p = p * t + 0.16928004f;
    const float q = size * (t * p) * __expf(-0.5f * g * g);
    return g < 0.0f ? -q : g - q;
}

// values = up * act(gate), in 32 bits, of the activations 0 silu, 1 gelu, 2 identity; 3: min(gate, limit) * sigmoid(1.702 min(gate, limit)) * (clamp(up, -limit,
// limit) + 1).  What is no number stays one.  The choice lies outside the loops, so that the values' exponentials and divisions overlap (inside, a gated product of 777
// tokens, 6912 x 1536, took 22.3 us).
template <int COUNT>
__device__ __forceinline__ void gated_values(const float (&up)[COUNT], const float (&gate)[COUNT], int activation, float limit, float (&values)[COUNT]) {
    if (activation == 0) {
#pragma unroll
        for (int i = 0; i < COUNT; ++i) values[i] = up[i] * __fdividef(gate[i], 1.0f + __expf(-gate[i]));
    } else if (activation == 1) {
#pragma unroll
        for (int i = 0; i < COUNT; ++i) values[i] = up[i] * gelu(gate[i]);
    } else if (activation == kSigmoidLimit) {
#pragma unroll
        for (int i = 0; i < COUNT; ++i) {
            const float g = at_most(gate[i], limit);
            values[i] = (at_most(at_least(up[i], -limit), limit) + 1.0f) * __fdividef(g, 1.0f + __expf(-kSigmoidLimitSlope * g));
        }
    } else {
#pragma unroll
        for (int i = 0; i < COUNT; ++i) values[i] = up[i] * gate[i];
    }
}

// Eight columns from `first` of a row of `width`, as float32, into v[at] on; past the width zeros.  VECTOR: the row starts on 16 bytes and the width is a multiple of 8.
template <bool VECTOR, int at = 0, typename T, int COUNT>
__device__ __forceinline__ void load_eight(const T* row, int first, int width, float (&v)[COUNT]) {
    if constexpr (VECTOR) {
        if (first >= width) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[at + i] = 0.0f;
        } else if constexpr (sizeof(T) == 2) {
            const uint4 raw = *reinterpret_cast<const uint4*>(row + first);
            const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[at + 2 * i] = __uint_as_float(words[i] << 16);
                v[at + 2 * i + 1] = __uint_as_float(words[i] & 0xffff0000u);
            }
        } else {
            const float4 low = *reinterpret_cast<const float4*>(row + first), high = *reinterpret_cast<const float4*>(row + first + 4);
            v[at + 0] = low.x, v[at + 1] = low.y, v[at + 2] = low.z, v[at + 3] = low.w, v[at + 4] = high.x, v[at + 5] = high.y, v[at + 6] = high.z, v[at + 7] = high.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[at + i] = first + i < width ? to_float(row[first + i]) : 0.0f;
    }
}

// Eight columns to `row`, rounded once; nothing past the width.
template <bool VECTOR, typename T>
__device__ __forceinline__ void store_eight(T* row, int first, int width, const float (&v)[8]) {
    if constexpr (VECTOR) {
        if (first >= width) return;
        if constexpr (sizeof(T) == 2) {
            uint4 raw;
            __nv_bfloat162* halves = reinterpret_cast<__nv_bfloat162*>(&raw);
#pragma unroll
            for (int i = 0; i < 4; ++i) halves[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
            *reinterpret_cast<uint4*>(row + first) = raw;
        } else {
            *reinterpret_cast<float4*>(row + first) = make_float4(v[0], v[1], v[2], v[3]);
            *reinterpret_cast<float4*>(row + first + 4) = make_float4(v[4], v[5], v[6], v[7]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (first + i < width) row[first + i] = from_float<T>(v[i]);
    }
}

}  // namespace lb
