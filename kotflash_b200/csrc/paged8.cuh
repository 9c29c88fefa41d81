// The 8-bit formats of paged K/V pools: codes with a power of two as the scale
// of each block of rows.  A scale is one byte, 127 + its exponent (e8m0), 255
// where the block stands for NaN; exponents lie within +-60.
//
// A floating code of 4 significant bits is as exact under any scale that keeps
// it off the subnormals, and a power of two makes everything around it exact:
// the value fits bf16 and fp16 as it is, reading back rounds nothing, and a
// block whose scale grows loses only the bits that fall off its codes.  An
// int8 code loses one bit at most to the scale's steps of two.
#pragma once
#include "kf_host.h"
#include "kf_sm100.cuh"

namespace kf {

constexpr int kMaxExponent = 60;  // (the sums of paged8_decode.cuh and their reciprocals rely on it)
constexpr int kNanScale = 255;

// Exponent of the smallest power of two that holds magnitudes up to x >= 0:
// x <= 448 2^e (e4m3), or x rounds to 127 2^e at most (int8); above
// kMaxExponent where there is none (infinities and NaN among them).
template <bool INT8>
KF_DEVI int scale_exponent(float x) {
  const uint32_t bits = __float_as_uint(x);
  const int e = (int)(bits >> 23) - 127;
  const uint32_t m = bits & 0x7fffffu;
  // 448 = 1.75 * 2^8; 127.5 = 1.9921875 * 2^6 would round to 128
  const int up = INT8 ? e - 6 + (m >= 0x7f0000u) : e - 8 + (m > 0x600000u);
  return up < -kMaxExponent ? -kMaxExponent : up;
}
KF_DEVI uint32_t scale_byte(int e) { return e > kMaxExponent ? kNanScale : (uint32_t)(127 + e); }
// Exponent of a stored scale (255: not asked).  Bytes that nobody stored count as the nearest.
KF_DEVI int scale_of_byte(uint32_t byte) { return min(max((int)byte - 127, -kMaxExponent), kMaxExponent); }
KF_DEVI float power2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }  // |e| <= 126

// Four values, already divided by their scale, to codes (to nearest, ties to even).
template <bool INT8>
KF_DEVI uint32_t encode4(float a, float b, float c, float d) {
  if constexpr (INT8) {
    const int x = __float2int_rn(a), y = __float2int_rn(b), z = __float2int_rn(c), w = __float2int_rn(d);
    return __byte_perm(__byte_perm(x, y, 0x0040), __byte_perm(z, w, 0x0040), 0x5410);
  } else {
    uint32_t r;
    asm("{\n\t.reg .b16 l, h;\n\tcvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n\t"
        "mov.b32 %0, {l, h};\n\t}"
        : "=r"(r)
        : "f"(a), "f"(b), "f"(c), "f"(d));
    return r;
  }
}

// Four codes as fp16 pairs: lo the first two, hi the others.  Exact.
template <bool INT8>
KF_DEVI void decode4(uint32_t codes, uint32_t& lo, uint32_t& hi) {
  if constexpr (INT8) {
    // 0x6400 | u is 1024 + u; with u = code + 128, less 1152 is the code
    codes ^= 0x80808080u;
    const uint32_t less = 0xe480e480u;  // -1152
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(__byte_perm(codes, 0x64646464u, 0x4140)), "r"(less));
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(hi) : "r"(__byte_perm(codes, 0x64646464u, 0x4342)), "r"(less));
  } else {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(codes));
  }
}
template <bool INT8>
KF_DEVI void decode4(uint32_t codes, float (&x)[4]) {
  uint32_t lo, hi;
  decode4<INT8>(codes, lo, hi);
  const float2 a = unpack2<false>(lo), b = unpack2<false>(hi);
  x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
}

// Elementwise maximum of two pairs of 16-bit magnitudes (of fp16 or bf16, by
// their bits: infinities and NaN are the largest).
KF_DEVI uint32_t max_magnitudes(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
KF_DEVI uint32_t magnitudes(uint4 w) {
  constexpr uint32_t M = 0x7fff7fffu;
  return max_magnitudes(max_magnitudes(w.x & M, w.y & M), max_magnitudes(w.z & M, w.w & M));
}
// The larger of the pair as fp32.
template <bool BF16>
KF_DEVI float largest(uint32_t pair) {
  return unpack2<BF16>(max(pair & 0xffffu, pair >> 16)).x;
}

// Eight 16-bit values times `by` to eight codes.
template <bool INT8, bool BF16>
KF_DEVI uint2 encode8(uint4 w, float by) {
  const float2 a = unpack2<BF16>(w.x), b = unpack2<BF16>(w.y), c = unpack2<BF16>(w.z), d = unpack2<BF16>(w.w);
  return make_uint2(encode4<INT8>(a.x * by, a.y * by, b.x * by, b.y * by),
                    encode4<INT8>(c.x * by, c.y * by, d.x * by, d.y * by));
}

// Checks what every entry point asks of a cache (before any launch).
int check_cache8(const char* what, const kf_paged8_cache& c);

// One launch of the attention kernel; args is a Paged8Args of paged8_decode.cuh.
struct Paged8Launch {
  const void* args;
  const CUtensorMap *map_k, *map_v;
  int steps;                       // 16-byte chunks of a row
  bool lines;                      // pages are brought as lines
  int rows, blocks;
  cudaStream_t stream;
};
int paged8_launch_e4m3_f16(const Paged8Launch& l);
int paged8_launch_e4m3_bf16(const Paged8Launch& l);
int paged8_launch_int8_f16(const Paged8Launch& l);
int paged8_launch_int8_bf16(const Paged8Launch& l);

}  // namespace kf
