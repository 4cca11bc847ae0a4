// Conversion of keys and values to what the cache stores: fp8 codes of the correctly rounded quotient
// x / scale, for the KV write kernels.
#pragma once

#include <type_traits>

#include "common.cuh"

namespace b200pa {

enum : int { kKvAuto = 0, kKvE4M3 = 1, kKvE5M2 = 2 };

// x / scale, correctly rounded, for one scale and many x.  The compiler's division spends a
// MUFU.RCP, a range check and a slow-path branch on every element, which made the KV write
// XU-bound; here the reciprocal is taken once and each quotient is the product x * r followed
// by two residual corrections q += fma(-q, s, x) * r.  The first leaves q within one ulp, the
// second then yields the correctly rounded quotient (Markstein's theorem; r is the correctly
// rounded reciprocal).  Used for positive scales within 2^+-60: there a residual can only
// lose bits to underflow for |x / s| < 2^-42, which is zero in both fp8 formats whatever its
// last bits are.  Other scales use the division.
struct ScaledDiv {
  float s, r;
  bool fast;
  uint64_t s2, nr2;  // {s, s} and {-r, -r} for the packed fp32 pipe
  __device__ __forceinline__ explicit ScaledDiv(float scale) : s(scale) {
    r = __fdiv_rn(1.f, scale);
    fast = scale >= 0x1p-60f && scale <= 0x1p60f;
    const float nr = -r;
    asm("mov.b64 %0, {%1, %1};" : "=l"(s2) : "f"(s));
    asm("mov.b64 %0, {%1, %1};" : "=l"(nr2) : "f"(nr));
  }
  // MINUS the two quotients, on the packed fp32 pipe (fma.rn.f32x2, sm_100).  The sequence
  // runs on the negated quotient q' = -x/s because that keeps the sign of a zero:
  //   q' = x * (-r);  e = fma(q', s, x) = x - q*s;  q' = fma(e, -r, q')
  // gives q' = -0 for x = +0 and +0 for x = -0, where the same steps on q itself turn -0
  // into +0.  The caller flips the sign bit of the fp8 codes instead (one XOR per four
  // codes).  An infinite or overflowing quotient comes out as NaN (inf - inf); the caller
  // sees its NaN code and redoes those elements with the division.
  // Callers check `fast` once per kernel, not per pair.
  __device__ __forceinline__ void neg_pair(float x0, float x1, float& o0, float& o1) const {
    asm("{\n"
        " .reg .b64 x, q, e;\n"
        " mov.b64 x, {%2, %3};\n"
        " mul.rn.f32x2 q, x, %4;\n"
        " fma.rn.f32x2 e, q, %5, x;\n"
        " fma.rn.f32x2 q, e, %4, q;\n"
        " fma.rn.f32x2 e, q, %5, x;\n"
        " fma.rn.f32x2 q, e, %4, q;\n"
        " mov.b64 {%0, %1}, q;\n"
        "}"
        : "=f"(o0), "=f"(o1)
        : "f"(x0), "f"(x1), "l"(nr2), "l"(s2));
  }
  __device__ __forceinline__ float operator()(float x) const {
    if (!fast) return __fdiv_rn(x, s);
    const float q0 = x * r;
    float q = fmaf(fmaf(-q0, s, x), r, q0);
    q = fmaf(fmaf(-q, s, x), r, q);
    const float a = fabsf(q0);
    return (a >= 0x1p-20f && a < 0x1p17f) ? q : q0;
  }
};

// Four 16-bit inputs (two 32-bit words of two elements each) -> four fp8 codes of MINUS the
// quotients x / s (ScaledDiv::neg_pair explains the sign), in one asm block so that the
// packed-fp32 register pairs are formed where the values are produced and no moves are
// needed around the packed instructions.
template <typename in_t, bool kE5M2>
__device__ __forceinline__ uint32_t neg_quant4(uint32_t w0, uint32_t w1, const ScaledDiv& div) {
  uint32_t out;
  if constexpr (std::is_same_v<in_t, __nv_bfloat16>) {
    if constexpr (kE5M2) {
      asm("{\n"
          " .reg .b32 a0, a1, b0, b1;\n"
          " .reg .b64 x, y, q, r, e;\n"
          " .reg .b16 lo, hi;\n"
          " shl.b32 a0, %1, 16;\n and.b32 a1, %1, 0xffff0000;\n"
          " shl.b32 b0, %2, 16;\n and.b32 b1, %2, 0xffff0000;\n"
          " mov.b64 x, {a0, a1};\n mov.b64 y, {b0, b1};\n"
          " mul.rn.f32x2 q, x, %3;\n mul.rn.f32x2 r, y, %3;\n"
          " fma.rn.f32x2 e, q, %4, x;\n fma.rn.f32x2 q, e, %3, q;\n"
          " fma.rn.f32x2 e, r, %4, y;\n fma.rn.f32x2 r, e, %3, r;\n"
          " fma.rn.f32x2 e, q, %4, x;\n fma.rn.f32x2 q, e, %3, q;\n"
          " fma.rn.f32x2 e, r, %4, y;\n fma.rn.f32x2 r, e, %3, r;\n"
          " mov.b64 {a0, a1}, q;\n mov.b64 {b0, b1}, r;\n"
          " cvt.rn.satfinite.e5m2x2.f32 lo, a1, a0;\n"
          " cvt.rn.satfinite.e5m2x2.f32 hi, b1, b0;\n"
          " mov.b32 %0, {lo, hi};\n"
          "}"
          : "=r"(out)
          : "r"(w0), "r"(w1), "l"(div.nr2), "l"(div.s2));
    } else {
      asm("{\n"
          " .reg .b32 a0, a1, b0, b1;\n"
          " .reg .b64 x, y, q, r, e;\n"
          " .reg .b16 lo, hi;\n"
          " shl.b32 a0, %1, 16;\n and.b32 a1, %1, 0xffff0000;\n"
          " shl.b32 b0, %2, 16;\n and.b32 b1, %2, 0xffff0000;\n"
          " mov.b64 x, {a0, a1};\n mov.b64 y, {b0, b1};\n"
          " mul.rn.f32x2 q, x, %3;\n mul.rn.f32x2 r, y, %3;\n"
          " fma.rn.f32x2 e, q, %4, x;\n fma.rn.f32x2 q, e, %3, q;\n"
          " fma.rn.f32x2 e, r, %4, y;\n fma.rn.f32x2 r, e, %3, r;\n"
          " fma.rn.f32x2 e, q, %4, x;\n fma.rn.f32x2 q, e, %3, q;\n"
          " fma.rn.f32x2 e, r, %4, y;\n fma.rn.f32x2 r, e, %3, r;\n"
          " mov.b64 {a0, a1}, q;\n mov.b64 {b0, b1}, r;\n"
          " cvt.rn.satfinite.e4m3x2.f32 lo, a1, a0;\n"
          " cvt.rn.satfinite.e4m3x2.f32 hi, b1, b0;\n"
          " mov.b32 %0, {lo, hi};\n"
          "}"
          : "=r"(out)
          : "r"(w0), "r"(w1), "l"(div.nr2), "l"(div.s2));
    }
  } else {
    const __half2 h0 = *reinterpret_cast<const __half2*>(&w0);
    const __half2 h1 = *reinterpret_cast<const __half2*>(&w1);
    float q0, q1, q2, q3;
    div.neg_pair(__low2float(h0), __high2float(h0), q0, q1);
    div.neg_pair(__low2float(h1), __high2float(h1), q2, q3);
    out = uint32_t(f32x2_to_fp8x2<kE5M2>(q0, q1)) | (uint32_t(f32x2_to_fp8x2<kE5M2>(q2, q3)) << 16);
  }
  return out;
}

// N consecutive elements.  fp8: four at a time - two pair conversions of the negated
// quotients, sign bits flipped back in the assembled word; a group of up to 16 codes that holds
// a NaN code (a NaN, or a quotient that overflowed inside neg_pair) is redone with the division,
// which is rare.
template <typename in_t, typename cache_t, int KV, int N>
__device__ __forceinline__ void convert_n(const in_t (&in)[N], cache_t* out, const ScaledDiv& div) {
  if constexpr (KV == kKvAuto) {
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = in[i];
  } else if constexpr (N % 4 == 0) {
    constexpr bool kE5 = KV == kKvE5M2;
    if (!div.fast) {  // the same for every thread of the launch
#pragma unroll
      for (int i = 0; i < N; ++i) out[i] = f32_to_fp8<kE5>(__fdiv_rn(to_f32(in[i]), div.s));
      return;
    }
    uint32_t w[N / 4];
    uint32_t nan_bits = 0;
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      uint32_t v;
      if constexpr (sizeof(in_t) == 2) {
        uint32_t w0, w1;
        const uint16_t b0 = *reinterpret_cast<const uint16_t*>(&in[i]);
        const uint16_t b1 = *reinterpret_cast<const uint16_t*>(&in[i + 1]);
        const uint16_t b2 = *reinterpret_cast<const uint16_t*>(&in[i + 2]);
        const uint16_t b3 = *reinterpret_cast<const uint16_t*>(&in[i + 3]);
        w0 = uint32_t(b0) | (uint32_t(b1) << 16);
        w1 = uint32_t(b2) | (uint32_t(b3) << 16);
        v = neg_quant4<in_t, kE5>(w0, w1, div);
      } else {
        float q0, q1, q2, q3;
        div.neg_pair(to_f32(in[i]), to_f32(in[i + 1]), q0, q1);
        div.neg_pair(to_f32(in[i + 2]), to_f32(in[i + 3]), q2, q3);
        v = uint32_t(f32x2_to_fp8x2<kE5>(q0, q1)) | (uint32_t(f32x2_to_fp8x2<kE5>(q2, q3)) << 16);
      }
      // a byte whose low seven bits are all ones is a NaN code in both formats
      nan_bits |= ((v & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
      w[i / 4] = v ^ 0x80808080u;
    }
    if (nan_bits != 0) {
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        uint32_t v = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          v |= uint32_t(f32_to_fp8<kE5>(__fdiv_rn(to_f32(in[i + k]), div.s))) << (8 * k);
        w[i / 4] = v;
      }
    }
#pragma unroll
    for (int i = 0; i < N / 4; ++i) reinterpret_cast<uint32_t*>(out)[i] = w[i];
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = f32_to_fp8<KV == kKvE5M2>(div(to_f32(in[i])));
  }
}

// The same conversion for 16-bit inputs that are already in registers as 32-bit words of two
// elements each (what 16-byte loads deliver): NW input words -> NW / 2 words of fp8 codes.  Works
// on the words directly, so nothing is unpacked into elements and packed again.
template <typename in_t, int KV, int NW>
__device__ __forceinline__ void convert_words(const uint32_t (&w)[NW], uint32_t (&out)[NW / 2],
                                              const ScaledDiv& div) {
  static_assert(sizeof(in_t) == 2 && KV != kKvAuto && NW % 2 == 0, "16-bit inputs, fp8 cache");
  constexpr bool kE5 = KV == kKvE5M2;
  auto slow4 = [&](uint32_t w0, uint32_t w1) -> uint32_t {
    const in_t* e0 = reinterpret_cast<const in_t*>(&w0);
    const in_t* e1 = reinterpret_cast<const in_t*>(&w1);
    return uint32_t(f32_to_fp8<kE5>(__fdiv_rn(to_f32(e0[0]), div.s))) |
           (uint32_t(f32_to_fp8<kE5>(__fdiv_rn(to_f32(e0[1]), div.s))) << 8) |
           (uint32_t(f32_to_fp8<kE5>(__fdiv_rn(to_f32(e1[0]), div.s))) << 16) |
           (uint32_t(f32_to_fp8<kE5>(__fdiv_rn(to_f32(e1[1]), div.s))) << 24);
  };
  if (!div.fast) {  // the same for every thread of the launch
#pragma unroll
    for (int i = 0; i < NW; i += 2) out[i / 2] = slow4(w[i], w[i + 1]);
    return;
  }
  uint32_t nan_bits = 0;
#pragma unroll
  for (int i = 0; i < NW; i += 2) {
    const uint32_t v = neg_quant4<in_t, kE5>(w[i], w[i + 1], div);
    nan_bits |= (v & 0x7F7F7F7Fu) + 0x01010101u;  // bit 7 of a byte: its low seven bits were all ones
    out[i / 2] = v ^ 0x80808080u;
  }
  if ((nan_bits & 0x80808080u) != 0) {
#pragma unroll
    for (int i = 0; i < NW; i += 2) out[i / 2] = slow4(w[i], w[i + 1]);
  }
}

}  // namespace b200pa
