// A cache of keys and values in 8 bits: how its numbers are held and how they lie in memory.
//
// A block is 16 tokens of one key/value head, and has a scale for its keys and one for its values: powers of two, held as 32-bit
// floats, the smallest 2^e (e in SCALE_LOW .. SCALE_HIGH) with 448 * 2^e at least as large as the block's largest magnitude. A number x is held
// as x 2^-e rounded to e4m3 (three bits behind the leading one, 448 the largest, none of it an infinity; infinities become NaN). So
// what is held, code * 2^e, is exact in bfloat16, and taking a block to a larger scale is exact but for numbers that fall below 2^-6 of it.
//
// In memory a page's blocks of a head lie together, and a block lies as the matrix instructions take it, so that a wave's 16-byte loads
// are operands as they arrive:
//   keys   [page][head][block of the page][head_size / 16][16 tokens][16 elements]
//   values [page][head][block of the page][head_size][16 tokens]
//   scales [page][head][block of the page], for either
// (a value is read along its tokens by the product with the softmax weights; held token by token, every load of it would have to be turned
// round through LDS.)
#pragma once

#include "common.h"

constexpr int BLOCK_TOKENS = 16;
constexpr int SCALE_LOW = -110, SCALE_HIGH = 118;   // 2^-9 * 2^-110 is no denormal of bfloat16, 448 * 2^118 below its largest
constexpr float CODE_LARGEST = 448.0f;
constexpr int SCALED_MAX_HEAD = 256;

typedef __attribute__((ext_vector_type(2))) float f32x2;

__device__ __forceinline__ float two_to(int e) { return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23); }   // e in -126 .. 127

// The e of a scale as it is held (whatever its bits are: it comes out inside the bounds).
__device__ __forceinline__ int scale_exponent(float scale) {
    return min(max((int)((__builtin_bit_cast(uint32_t, scale) >> 23) & 255u) - 127, SCALE_LOW), SCALE_HIGH);
}

// The e that a largest magnitude needs (0: the smallest): with largest = m 2^x, 1 <= m < 2, it is x - 8, and one more where m > 1.75.
__device__ __forceinline__ int needed_exponent(float largest) {
    const uint32_t bits = __builtin_bit_cast(uint32_t, largest);
    return min(max((int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0), SCALE_LOW), SCALE_HIGH);
}

// A number's magnitude as it counts for its block's scale: infinities and NaN do not.
__device__ __forceinline__ float counted_magnitude(float x) {
    const uint32_t bits = __builtin_bit_cast(uint32_t, x) & 0x7fffffffu;
    return bits >= 0x7f800000u ? 0.0f : __builtin_bit_cast(float, bits);
}

// x times the scale's inverse, as the conversion to 8 bits takes it.
__device__ __forceinline__ float ready_for_code(float x, float inverse) {
    const float scaled = fminf(fmaxf(x * inverse, -CODE_LARGEST), CODE_LARGEST);
    return (__builtin_bit_cast(uint32_t, x) & 0x7f800000u) == 0x7f800000u ? __builtin_nanf("") : scaled;
}

// Four numbers to four codes, and two.
__device__ __forceinline__ uint32_t four_codes(float a, float b, float c, float d) {
    int packed = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, packed, true);
}

// Four codes taken to a scale 1 / factor times theirs.
__device__ __forceinline__ uint32_t rescaled_codes(uint32_t codes, float factor) {
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, true);
    return four_codes(lo[0] * factor, lo[1] * factor, hi[0] * factor, hi[1] * factor);
}

// Eight codes times a scale, as an operand of the matrix instructions: exact.
__device__ __forceinline__ bf16x8 eight_numbers(uint32_t lo, uint32_t hi, float scale) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// The high bit of every byte of four codes that are no number (s1111111).
__device__ __forceinline__ uint32_t not_numbers(uint32_t codes) { return ((codes & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// Rows of a call that fall into one block are a run where they are neighbours and their slots follow each other. Lane i of a wave looks at row `from` + i (32 of them are
// enough: a run has at most 16 rows), whose slot is left in `slot`; the bits of the result are the rows that begin a run, rows behind the last among them. Rows
// that go nowhere (their slots are negative, or lie behind the pages) are runs of their own, as many neighbours as up to the next multiple of 16.
__device__ __forceinline__ uint32_t run_begins(const int* __restrict__ slots, int from, int n_rows, long long n_slots, int lane, int& slot) {
    const int row = from + (lane & 31), here = min(row, n_rows - 1);
    slot = slots[here];
    const int before = slots[max(here - 1, 0)];
    const bool nowhere = slot < 0 || slot >= n_slots, before_nowhere = before < 0 || before >= n_slots;
    const bool follows = nowhere ? row % BLOCK_TOKENS != 0 : slot / BLOCK_TOKENS == before / BLOCK_TOKENS && slot == before + 1;
    return (uint32_t)__ballot(row <= 0 || row >= n_rows || nowhere != before_nowhere || !follows);
}
