// The 4-bit form of cached keys and values and of weights, shared by the kernels that write, read and multiply it.
//
// ``group`` neighbouring values share a minimum z and a step s, both float16; a value is c s + z with a code c of 0 .. 15:
//   z = float16(min x),  s = float16(max(max x - z, 0) f) with f the float32 next to 1/15, the difference and the product in float32,
//   c = (x - z) / s rounded to the nearest (ties to even) and cut to 0 .. 15;  s = 0 gives c = 0.
// A group that holds a value beyond 60,000, or one that is not finite, becomes not a number as a whole (s = z = NaN): c s + z of every
// other group is a finite float16 after rounding.
//
// Codes are laid out for the matrix instructions that read them (mma.sync m16n8k16, float16): a 32-bit word w holds 8 codes that lie
// together along the axis a lane reads, and
//   w & 0x000f000f          is the float16 pair (c0, c4) 2^-24      (float16 numbers below 2^-14 have the fixed step 2^-24:
//   w & 0x00f000f0          is the float16 pair (c1, c5) 2^-20       a small integer IS its own bit pattern)
//   (w >> 8) & 0x000f000f   is (c2, c6) 2^-24, and so on:
// five instructions turn 8 codes into operands, exactly and without a bias to take off again; the powers of two go into the other
// operand and into the sums.  (Codes or'ed into the mantissa of 1024, the usual way, cost one more instruction a pair to take the 1024
// off.)
//
// A tile: 16 tokens of one KV head (cache), or 16 rows of a weight by 64 columns.
//   K codes   block b of 64 channels, lane (r, l) = 4 r + l: words of channels 64 b + 8 l .. + 8 (first half of the block) and
//             64 b + 32 + 8 l .. + 8 (second half), tokens r and r + 8: 16 bytes a lane, 512 a block
//   V codes   block b, lane (r, l): words of tokens 2 l, 2 l + 1, 2 l + 8, 2 l + 9; codes 0 .. 3 of a word are channels
//             64 b + 4 r .. + 4, codes 4 .. 7 channels 64 b + 32 + 4 r .. + 4
//   (s, z) of K, token by token and group by group, then those of V
// A weight's tile has codes as K's and its (s, z) row by row; rows 0 .. 7 of a gated weight's tile are gate rows, 8 .. 15 the up rows that belong
// to them, so that a lane's sums (rows r and r + 8) are the two halves of its results.
#pragma once
#include "common.cuh"
#include <cuda_fp16.h>
#include <type_traits>

#define I4_LIMIT 60000.0f

__host__ __device__ constexpr int i4_cache_tile_bytes(int d, int group) { return 16 * d + 128 * (d / group); }
__host__ __device__ constexpr int i4_weight_tile_bytes(int group) { return 512 + 64 * (64 / group); }       // group 32 or 64

// byte offsets inside a tile
__device__ __forceinline__ int i4_k_word(int token, int channel) {
    const int b = channel >> 6, half = (channel >> 5) & 1, l = (channel >> 3) & 3;
    return b * 512 + (4 * (token & 7) + l) * 16 + (half * 2 + (token >> 3)) * 4;
}
__device__ __forceinline__ int i4_v_word(int d, int token, int b, int r) {
    return 8 * d + b * 512 + (4 * r + ((token & 7) >> 1)) * 16 + ((token & 1) + 2 * (token >> 3)) * 4;
}
__device__ __forceinline__ int i4_k_step(int d, int groups, int token, int g) { return 16 * d + (token * groups + g) * 4; }
__device__ __forceinline__ int i4_v_step(int d, int groups, int token, int g) { return 16 * d + 64 * groups + (token * groups + g) * 4; }

// (s, z) of a group with the extremes lo and hi; ok: all its values are finite and at most I4_LIMIT.  Where rounding takes z above hi (float32
// groups that are nearly constant), s is 0, as for any group of one value: attention scales its weights by the largest step it meets.
__device__ __forceinline__ __half2 i4_step(float lo, float hi, bool ok) {
    const __half z = __float2half_rn(lo);
    const __half s = __float2half_rn(__fmul_rn(fmaxf(__fsub_rn(hi, __half2float(z)), 0.0f), 1.0f / 15.0f));
    return ok ? __halves2half2(s, z) : __halves2half2(__ushort_as_half(0x7e00), __ushort_as_half(0x7e00));
}
// The code of x.  (x - z) / s in float32 is off by less than 2^-18 (both factors rounded, the quotient below 16): where it lies that near to the
// border between two codes, the border itself decides, in float64, where (x - z) and (n + 1/2) s have room.
__device__ __forceinline__ unsigned i4_code(float x, float s, float z, float inv) {
    const float t = (x - z) * inv;
    const float below = floorf(t), rest = t - below;
    float c = rest > 0.5f ? below + 1.0f : below;
    if (fabsf(rest - 0.5f) < 1.0f / 4096.0f) {
        const double d = (double)x - (double)z, border = ((double)below + 0.5) * (double)s;
        const bool odd = ((int)below & 1) != 0;
        c = d > border || (d == border && odd) ? below + 1.0f : below;
    }
    return (unsigned)fminf(fmaxf(c, 0.0f), 15.0f);        // a step of NaN or 0 comes with inv 0: code 0
}
__device__ __forceinline__ float i4_inverse(float s) { return s > 0.0f ? 1.0f / s : 0.0f; }

// (not volatile: the products are functions of their operands, and the compiler may order them)
__device__ __forceinline__ void i4_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the first product of a chain: nothing to add to
__device__ __forceinline__ void i4_mma_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("{\n.reg .f32 z;\nmov.f32 z, 0f00000000;\n"
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {z,z,z,z};\n}"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t i4_smem(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ uint32_t i4_arrived(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}"
                 : "=r"(ok) : "r"(i4_smem(bar)), "r"(parity) : "memory");
    return ok;
}
// A lane's wait for a barrier's phase, with a limit: the thread sleeps in the instruction itself.
__device__ __forceinline__ bool i4_wait(uint64_t* bar, uint32_t parity) {
    for (uint32_t i = 0; i < (1u << 16); ++i)
        if (i4_arrived(bar, parity)) return true;
    return false;
}
// A whole warp's: its lanes leave together.
__device__ __forceinline__ bool i4_warp_wait(uint64_t* bar, uint32_t parity) {
    for (uint32_t i = 0; i < (1u << 16); ++i)
        if (__all_sync(0xffffffffu, i4_arrived(bar, parity))) return true;
    return false;
}
// A run of bytes into shared memory, counted on the barrier (both addresses and the size in multiples of 16); one lane calls it.
__device__ __forceinline__ void i4_copy(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(i4_smem(bar)), "r"(bytes) : "memory");
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(i4_smem(dst)), "l"(src), "r"(bytes), "r"(i4_smem(bar)) : "memory");
}

// Four of a word's codes as operands (SHIFT 0 or 8): the even pair and the odd one, which is 16 times too large.  Plain: the bits of the codes,
// float16 numbers of 2^-24.  CENTRED: codes less 8 as ordinary float16 numbers, which the float32 path takes for two instructions a word more:
// tensor cores cut what they add to a sum, all the earlier where the operands are float16 numbers below 2^-14, and sums of codes that are all
// positive lose, next to a result that their minimum's part nearly cancels, more of the bits that float32 is asked for.  (Attention of 4 x 700
// keys, float32, off by 2.6e-5 of the result with the plain codes, 5.9e-6 with codes less 8 below 2^-14.)
template <bool CENTRED> constexpr float i4_unit = CENTRED ? 1.0f : 0x1p24f;       // what a sum of products with the codes is multiplied by
template <bool CENTRED, int SHIFT>
__device__ __forceinline__ void i4_pairs(uint32_t w, uint32_t& even, uint32_t& odd) {
    even = (w >> SHIFT) & 0x000f000fu;
    odd = (w >> SHIFT) & 0x00f000f0u;
    if (CENTRED) {
        even |= 0x64006400u;                          // 1024 + c
        odd |= 0x64006400u;                           // 1024 + 16 c
        const uint32_t e8 = 0x64086408u, o8 = 0x64806480u;        // 1024 + 8, 1024 + 16 * 8
        __half2 e = __hsub2(*reinterpret_cast<__half2*>(&even), *reinterpret_cast<const __half2*>(&e8));
        __half2 o = __hsub2(*reinterpret_cast<__half2*>(&odd), *reinterpret_cast<const __half2*>(&o8));
        even = *reinterpret_cast<uint32_t*>(&e);
        odd = *reinterpret_cast<uint32_t*>(&o);
    }
}
// (s, z) as float32; CENTRED: z is the value of code 8
template <bool CENTRED>
__device__ __forceinline__ float2 i4_step_of(uint32_t v) {
    float2 f = __half22float2(*reinterpret_cast<__half2*>(&v));
    if (CENTRED) f.y = fmaf(8.0f, f.x, f.y);
    return f;
}
__device__ __forceinline__ float i4_relu(float v) { return v < 0.0f ? 0.0f : v; }        // NaN stays
// the smaller one; NaN where either is
__device__ __forceinline__ float i4_min(float a, float b) {
    float v;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(v) : "f"(a), "f"(b));
    return v;
}
__device__ __forceinline__ uint32_t i4_pack(float lo, float hi) {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ float2 i4_unpack(uint32_t v) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }

// What a row's scores are multiplied by, kept within float32's normal numbers: beyond them (queries of 2^117 and more, tiny ones beside tiny scales)
// scores are as far apart, or as near, as makes no difference to a softmax, while infinity and 0 would make NaN of scores that are 0 or hidden.
// (Comparisons: NaN stays.)
__device__ __forceinline__ float i4_normal(float v) { return v > 0x1.fffffep127f ? 0x1.fffffep127f : v < 0x1p-126f ? 0x1p-126f : v; }
// The power of two that brings a row's largest magnitude into [2^14, 2^15): a float16 then holds bfloat16 values exactly down to 2^-30 of the
// largest, and a 16th of them (for codes that come 16 times too large) down to 2^-27.  Its bits are those of 2^14 less the largest's exponent; 1 for a row of zeros, NaN for one that is not finite.
__device__ __forceinline__ float i4_row_scale(float largest) {
    if (!(largest <= 3.402823466e38f)) return __int_as_float(0x7fc00000);
    const int e = (int)(__float_as_uint(largest) >> 23) - 127;          // subnormal numbers count as 2^-127
    const int k = min(14 - e, 126);
    return largest == 0.0f ? 1.0f : __uint_as_float((uint32_t)(k + 127) << 23);
}
