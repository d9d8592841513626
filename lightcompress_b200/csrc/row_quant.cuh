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

// ---- rows in registers ---------------------------------------------------------------------------------------
// kWarps warps hold a row, kVecs 16-byte vectors a lane; one warp to a row needs no barrier, and a CTA then holds
// eight rows.
template <int kWarps>
struct RowGroup {
  static constexpr int kRows = kWarps == 1 ? 8 : 1;            // rows of a CTA
  static constexpr int kThreads = kWarps == 1 ? 256 : kWarps * 32;
  static constexpr int kLanes = kWarps * 32;                   // threads of a row
  __device__ __forceinline__ static int row() { return kWarps == 1 ? threadIdx.x >> 5 : 0; }
  __device__ __forceinline__ static int lane() { return kWarps == 1 ? threadIdx.x & 31 : threadIdx.x; }

  // The sum of v over the row's threads, the same in all of them.  red: kWarps floats of shared memory that no other
  // reduction of this CTA uses (each call site has its own, so that one barrier a call is enough).
  __device__ __forceinline__ static float sum(float v, float* red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (kWarps == 1) return v;
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    float s = red[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) s += red[w];
    return s;
  }
  // min and max likewise; red: 2 * kWarps floats
  __device__ __forceinline__ static void range(float& mn, float& mx, float* red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      mx = nan_max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      mn = nan_min(mn, __shfl_xor_sync(0xffffffffu, mn, o));
    }
    if (kWarps == 1) return;
    if ((threadIdx.x & 31) == 0) {
      red[threadIdx.x >> 5] = mx;
      red[kWarps + (threadIdx.x >> 5)] = mn;
    }
    __syncthreads();
    mx = red[0];
    mn = red[kWarps];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) {
      mx = nan_max(mx, red[w]);
      mn = nan_min(mn, red[kWarps + w]);
    }
  }
};

// both forms from a row's minimum and maximum (zero included): max |v| is the larger of the two magnitudes
__device__ __forceinline__ RowQuant row_quant_of(float mn, float mx, bool sym) {
  return sym ? row_quant<true>(0.f, nan_max(mx, -mn)) : row_quant<false>(mn, mx);
}

// the codes of N (1, 2, 4 or 8) neighbouring values, stored at p (N-byte aligned)
template <int N>
__device__ __forceinline__ void store_row_codes(int8_t* p, const float (&v)[N], const RowQuant& q, bool sym) {
  if constexpr (N == 1) {
    *p = q.bad ? (int8_t)0 : (int8_t)(sym ? row_code<true>(v[0], q) : row_code<false>(v[0], q));
    return;
  } else if constexpr (N == 2) {
    const int c0 = sym ? row_code<true>(v[0], q) : row_code<false>(v[0], q);
    const int c1 = sym ? row_code<true>(v[1], q) : row_code<false>(v[1], q);
    *reinterpret_cast<char2*>(p) = q.bad ? make_char2(0, 0) : make_char2((signed char)c0, (signed char)c1);
  } else {
  uint32_t w[N / 4];
#pragma unroll
  for (int j = 0; j < N / 4; ++j) {
    if (q.bad) {
      w[j] = 0u;
    } else if (sym) {
      w[j] = pack4(row_code<true>(v[4 * j], q), row_code<true>(v[4 * j + 1], q), row_code<true>(v[4 * j + 2], q),
                   row_code<true>(v[4 * j + 3], q));
    } else {
      w[j] = pack4(row_code<false>(v[4 * j], q), row_code<false>(v[4 * j + 1], q), row_code<false>(v[4 * j + 2], q),
                   row_code<false>(v[4 * j + 3], q));
    }
  }
  if (N == 4) *reinterpret_cast<uint32_t*>(p) = w[0];
  else *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[N / 4 - 1]);
  }
}

// N neighbouring values as they lie in memory: a 16-byte vector, held as four whole registers, or two values or one where
// rows are not aligned to more (a warp still reads 64 to 256 contiguous bytes at once).
template <typename T, int N> struct RawOf { typedef uint4 type; };
template <typename T> struct RawOf<T, 1> { typedef T type; };
template <typename T> struct RawOf<T, 2> { typedef uint32_t type; };
template <> struct RawOf<float, 2> { typedef uint2 type; };
template <typename T, int N> using Raw = typename RawOf<T, N>::type;

template <typename T, int N>
__device__ __forceinline__ Raw<T, N> load_stream(const T* p) {             // read once
  if constexpr (N == 1) return *p;
  else return __ldcs(reinterpret_cast<const Raw<T, N>*>(p));
}
template <typename T, int N>
__device__ __forceinline__ void unpack(const Raw<T, N>& r, float (&f)[N]) {
  if constexpr (N == 1) {
    f[0] = Elem<T>::to_f(r);
  } else {
    const T* p = reinterpret_cast<const T*>(&r);
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = Elem<T>::to_f(p[i]);
  }
}
template <typename T, int N>
__device__ __forceinline__ Raw<T, N> pack(const float (&f)[N]) {
  if constexpr (N == 1) {
    return Elem<T>::from_f(f[0]);
  } else {
    Raw<T, N> r;
    T* p = reinterpret_cast<T*>(&r);
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = Elem<T>::from_f(f[i]);
    return r;
  }
}

// Which kernel holds rows of `vecs` 16-byte vectors: f(RowShape<warps of a row, vectors a lane>); false where none does.
// One warp to a row up to 2 KB, which needs no barrier; above, the fewest warps whose registers still leave several CTAs to
// an SM (4096 values in bf16, 8192 rows: 4 x 4 14.7 us, 8 x 2 17.5, 16 x 1 27.4; 11008 values, quantised: 8 x 6 20.1, 16 x 3
// 28.9; norms, with two inputs: 108 and 69).  A few rows leave the SMs empty: there what counts is how little a
// lane does.  Not so for norms: a sum's association follows the shape, and a row's result
// must not depend on how many others there are (one row of 4096: 3.2 us instead of 2.7).
template <int W, int V> struct RowShape {
  static constexpr int kWarps = W, kVecs = V;
};
template <bool kNorm, typename F>
bool with_row_shape(int64_t vecs, int64_t rows, F&& f) {
  const bool few = !kNorm && rows <= kNumSMsB200;
  if (vecs <= 32) f(RowShape<1, 1>{});
  else if (vecs <= 64) f(RowShape<1, 2>{});
  else if (vecs <= 128) f(RowShape<1, 4>{});
  else if (vecs <= 256) f(RowShape<4, 2>{});
  else if (vecs <= 512 && few) f(RowShape<8, 2>{});
  else if (vecs <= 512) f(RowShape<4, 4>{});
  else if (vecs <= 1024 && few) f(RowShape<16, 2>{});
  else if (vecs <= 1024) f(RowShape<8, 4>{});
  else if (vecs <= 1536 && (few || kNorm)) f(RowShape<16, 3>{});
  else if (vecs <= 1536) f(RowShape<8, 6>{});
  else if (vecs <= 2048 && kNorm) f(RowShape<8, 8>{});
  else if (vecs <= 2048) f(RowShape<16, 4>{});
  else if (vecs <= 4096) f(RowShape<16, 8>{});
  else return false;
  return true;
}
// The same for rows of pairs or single values, where what takes long is how many small accesses a lane makes (norms of 19
// rows of 4092 in bf16: 3.9 us by pairs, 5.6 by single values; 2048 rows of 4094: 14.8 and 20.6; 10 rows of 1794 quantised
// on 8 x 4 1.5, on 4 x 16 1.9).
template <bool kNorm, typename F>
bool with_value_shape(int64_t units, int64_t rows, F&& f) {
  const bool few = !kNorm && rows <= kNumSMsB200;
  if (units <= 128) f(RowShape<1, 4>{});
  else if (units <= 512) f(RowShape<4, 4>{});
  else if (units <= 1024 && few) f(RowShape<8, 4>{});
  else if (units <= 1024) f(RowShape<4, 8>{});
  else if (units <= 2048 && few) f(RowShape<16, 4>{});
  else if (units <= 2048) f(RowShape<8, 8>{});
  else if (units <= 4096 && few) f(RowShape<16, 8>{});
  else if (units <= 4096) f(RowShape<8, 16>{});
  else if (units <= 8192) f(RowShape<16, 16>{});
  else if (units <= 16384) f(RowShape<16, 32>{});
  else return false;
  return true;
}

}  // namespace lc
