// 8-bit integer quantisation of one row (token), shared by the kernels that produce a row and quantise it.
//
//   symmetric   a = max(max |v|, 1e-5);               s = a / 127, r = 127 * (1 / a), z = 0,  q = rint(v r)
//   asymmetric  lo = min(min v, 0), hi = max(max v, 0), d = max(hi - lo, 1e-5);
//               s = d / 255, r = 255 * (1 / d), z = -128 - rint(lo r),  q = clamp(rint(v r) + z, -128, 127)
//
// s and r are fp32 numbers, each operation of theirs rounded to nearest; v r is rounded once, to the nearest integer
// with ties to even: fma(v, r, 1.5 * 2^23) leaves rint(v r) in the low bits of its result, so an element costs one
// FFMA and its share of a byte pack instead of a division.  |v r| <= 255.0001, far inside the trick's range.
// A row with a NaN or an infinity (or, asymmetric, one whose hi - lo overflows) gets s = NaN and codes 0.
#pragma once

#include <float.h>

#include "lc_common.cuh"

namespace lc {

constexpr float kRintMagic = 12582912.f;        // 1.5 * 2^23
constexpr int kRintBias = 0x4B400000;           // its bits

struct RowQuant {
  float r, s;
  int z;
  bool bad;
};

// sym: mx = max |v|, mn unused.  asym: mn = min v, mx = max v (either may lie on the wrong side of zero).
template <bool kSym>
__device__ __forceinline__ RowQuant row_quant(float mn, float mx) {
  RowQuant q;
  float wide;
  if (kSym) {
    wide = nan_max(mx, 1e-5f);
  } else {
    mn = nan_min(mn, 0.f);
    wide = nan_max(__fsub_rn(nan_max(mx, 0.f), mn), 1e-5f);
  }
  q.bad = !(wide <= FLT_MAX);
  constexpr float steps = kSym ? 127.f : 255.f;
  q.s = q.bad ? __int_as_float(0x7fffffff) : __fdiv_rn(wide, steps);
  q.r = q.bad ? 0.f : __fmul_rn(steps, __frcp_rn(wide));
  q.z = (kSym || q.bad) ? 0 : -128 - (__float_as_int(__fmaf_rn(mn, q.r, kRintMagic)) - kRintBias);
  return q;
}

// the code of one value as an integer whose low byte is the int8 code
template <bool kSym>
__device__ __forceinline__ int row_code(float v, const RowQuant& q) {
  const int t = __float_as_int(__fmaf_rn(v, q.r, kRintMagic));
  if (kSym) return t;                                  // 0x4B400000 + rint: the low byte is the code
  return min(127, max(-128, t - kRintBias + q.z));
}

__device__ __forceinline__ uint32_t pack4(int a, int b, int c, int d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// what a thread keeps of the values it has seen
template <bool kSym>
struct RowRange {
  float mn = 0.f, mx = 0.f;      // zero belongs to the range either way
  __device__ __forceinline__ void add(float v) {
    if (kSym) {
      mx = nan_max(mx, fabsf(v));
    } else {
      mx = nan_max(mx, v);
      mn = nan_min(mn, v);
    }
  }
  __device__ __forceinline__ void warp_reduce() {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      mx = nan_max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      if (!kSym) mn = nan_min(mn, __shfl_xor_sync(0xffffffffu, mn, o));
    }
  }
};

}  // namespace lc
