// Per-token 8-bit quantisation of activations in front of the integer linear (the scaled_int8_quant call of
// the reference's VllmQuantLinearInt8, llmc/compression/quantization/module_utils.py:145-166), of a tensor or of
// the gated activation act(gate) * up that feeds an MLP's down projection.  Arithmetic: row_quant.cuh.
#include <type_traits>

#include "row_quant.cuh"

namespace lc {
namespace {

constexpr int kThreads = 256;

enum Act { kNone = 0, kSilu = LC_ACT_SILU, kGelu = LC_ACT_GELU, kGeluTanh = LC_ACT_GELU_TANH };

// Quotients and exponentials by the fast intrinsics.  __expf(y) is off by up to (2 + 1.17 |y|) 2^-23 relative, a quotient by
// two steps.  What comes out is off relative to itself, in the negative tail as well, because a token whose gates all lie
// there takes its scale from it:
//   silu       x / (1 + e^-x)                                                          (5 + 1.2 |x|) 2^-23
//   gelu_tanh  x / (1 + e^-u), u = 2 sqrt(2 / pi) (x + 0.044715 x^3), seven roundings   (5 + 4.7 |u|) 2^-23
//   gelu       x - x q or, below zero, x q: q = erfc(|x| / sqrt 2) / 2 = t P(t) e^(-x^2 / 2), t = 1 / (1 + 0.27 |x|), P of degree
//              6 fitted to the least relative error (1.5e-6 for |x| < 20, its roundings included)   (18 + 0.9 x^2) 2^-23
// A thousandth of a code is 2^-17: silu down to -49, gelu_tanh to -4.3, gelu to -7; twice that gelu_tanh to -6.1, gelu to -11.
// Where e^-x, e^-u or e^(x^2 / 2) leaves 2^126 (below -87, -10 and -13) the value is under 2^-119 and taken as zero.  The library's erff and tanhf bound the kernel: 40 and 36 us for 2048 x 11008 in bf16.  (A polynomial for erfc with a
// bound on its absolute error alone costs two steps less, 29 us where this one takes 31, and is off by a hundredth of the value
// at -8; an exponential whose error does not grow with its argument costs silu 25 us instead of 21.5.)
template <int kAct>
__device__ __forceinline__ float act_of(float x) {
  if (kAct == kSilu) return __fdividef(x, 1.f + __expf(-x));
  if (kAct == kGeluTanh) return __fdividef(x, 1.f + __expf(-1.5957691216057308f * (x + 0.044715f * x * x * x)));
  if (kAct == kGelu) {
    const float t = __fdividef(1.f, fmaf(0.27f, fabsf(x), 1.f));
    float p = -0.0610578172f;
    p = fmaf(p, t, 0.159365267f), p = fmaf(p, t, -0.0255874731f), p = fmaf(p, t, 0.118717268f);
    p = fmaf(p, t, 0.0923243687f), p = fmaf(p, t, 0.108561143f), p = fmaf(p, t, 0.107676633f);
    const float xq = x * (p * t * __expf(-0.5f * x * x));
    return x >= 0.f ? x - xq : xq;
  }
  return x;
}

struct QuantArgs {
  const void* x;        // gate when an activation is given
  const void* up;
  int64_t rows, cols, ldx, ldu, ldc;
  int8_t* codes;
  float* scales;
  int32_t* zeros;       // NULL: symmetric
};

template <bool kSym>
__device__ __forceinline__ RowQuant block_row_quant(RowRange<kSym> m, float* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  m.warp_reduce();
  __syncthreads();                       // red may still be read for the previous row
  if (lane == 0) {
    red[warp] = m.mx;
    red[8 + warp] = m.mn;
  }
  __syncthreads();
  float mx = red[0], mn = red[8];
#pragma unroll
  for (int w = 1; w < kThreads / 32; ++w) {
    mx = nan_max(mx, red[w]);
    mn = nan_min(mn, red[8 + w]);
  }
  return row_quant<kSym>(mn, mx);
}

// Any width and alignment: a CTA per row, the row read twice.
template <typename T, int kAct, bool kSym>
__global__ void __launch_bounds__(kThreads) quant_any_kernel(QuantArgs a) {
  using E = Elem<T>;
  __shared__ float red[16];
  begin_dependent();
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    const T* u = static_cast<const T*>(a.up) + row * a.ldu;
    auto value = [&](int64_t c) {
      const float v = E::to_f(x[c]);
      return kAct == kNone ? v : act_of<kAct>(v) * E::to_f(u[c]);
    };
    RowRange<kSym> m;
    for (int64_t c = threadIdx.x; c < a.cols; c += kThreads) m.add(value(c));
    const RowQuant q = block_row_quant<kSym>(m, red);
    int8_t* out = a.codes + row * a.ldc;
    for (int64_t c = threadIdx.x; c < a.cols; c += kThreads)
      out[c] = q.bad ? (int8_t)0 : (int8_t)row_code<kSym>(value(c), q);
    if (threadIdx.x == 0) {
      a.scales[row] = q.s;
      if (!kSym) a.zeros[row] = q.z;
    }
  }
}

// Rows that registers hold, by 16-byte vectors or, less aligned, by pairs or single values: read once, written once.
// HBM-bound: 16384 x 11008 in bf16 84 us (6.4 TB/s, 98 % of a copy's rate), with a zero point 92; silu(gate) * up 147 (6.1
// TB/s), the tanh form of gelu 156, the erf form 219, the last two bound by their arithmetic.
template <typename T, int N, int kWarps, int kVecs, int kAct>
__global__ void __launch_bounds__(RowGroup<kWarps>::kThreads) quant_rows_kernel(QuantArgs a) {
  using G = RowGroup<kWarps>;
  constexpr bool kGated = kAct != kNone;
  __shared__ float red[2 * kWarps];
  begin_dependent();
  const int64_t row = (int64_t)blockIdx.x * G::kRows + G::row();
  if (G::kRows > 1 && row >= a.rows) return;                           // a whole warp, and no barrier follows
  const int vecs = (int)(a.cols / N);
  const bool sym = a.zeros == nullptr;
  const T* x = static_cast<const T*>(a.x) + row * a.ldx;
  const T* u = static_cast<const T*>(a.up) + row * a.ldu;
  Raw<T, N> rx[kVecs], ru[kGated ? kVecs : 1];
#pragma unroll
  for (int k = 0; k < kVecs; ++k) {
    const int i = G::lane() + k * G::kLanes;
    if constexpr (!kGated) {
      rx[k] = i < vecs ? load_stream<T, N>(x + i * N) : pack<T, N>({});
    } else if (i < vecs) {                                             // a vector that is not there costs no activation
      rx[k] = load_stream<T, N>(x + i * N);
      ru[k] = load_stream<T, N>(u + i * N);
    }
  }
  float v[kVecs][N];
  float mn = 0.f, mx = 0.f;
#pragma unroll
  for (int k = 0; k < kVecs; ++k) {
    if (!kGated || G::lane() + k * G::kLanes < vecs) {
      unpack<T, N>(rx[k], v[k]);
      if (kGated) {
        float w[N];
        unpack<T, N>(ru[k], w);
#pragma unroll
        for (int j = 0; j < N; ++j) v[k][j] = act_of<kAct>(v[k][j]) * w[j];
      }
#pragma unroll
      for (int j = 0; j < N; ++j) {
        mx = nan_max(mx, v[k][j]);
        mn = nan_min(mn, v[k][j]);
      }
    }
  }
  G::range(mn, mx, red);
  const RowQuant q = row_quant_of(mn, mx, sym);
  int8_t* out = a.codes + row * a.ldc;
#pragma unroll
  for (int k = 0; k < kVecs; ++k) {
    const int i = G::lane() + k * G::kLanes;
    if (i < vecs) store_row_codes<N>(out + i * N, v[k], q, sym);
  }
  if (G::lane() == 0) {
    a.scales[row] = q.s;
    if (!sym) a.zeros[row] = q.z;
  }
}

// whether quant_rows_kernel took the rows
template <typename T, int kAct>
bool launch_rows(const QuantArgs& a, cudaStream_t st) {
  constexpr int N = Elem<T>::kPerVec;
  if (a.rows > 0x7fffffff) return false;
  // whether every row begins at a multiple of n values
  auto by = [&](int n) {
    return a.cols % n == 0 && (a.rows == 1 || (a.ldx % n == 0 && a.ldu % n == 0 && a.ldc % n == 0)) &&
           reinterpret_cast<uintptr_t>(a.x) % (n * sizeof(T)) == 0 && reinterpret_cast<uintptr_t>(a.up) % (n * sizeof(T)) == 0 &&
           reinterpret_cast<uintptr_t>(a.codes) % n == 0;
  };
  auto go = [&](auto shape, auto width) {
    using S = decltype(shape);
    using G = RowGroup<S::kWarps>;
    launch_dependent(quant_rows_kernel<T, decltype(width)::value, S::kWarps, S::kVecs, kAct>,
                     dim3((unsigned)((a.rows + G::kRows - 1) / G::kRows)), G::kThreads, 0, st, a);
  };
  if (by(N)) return with_row_shape<false>(a.cols / N, a.rows, [&](auto s) { go(s, std::integral_constant<int, N>{}); });
  if (by(2)) return with_value_shape<false>(a.cols / 2, a.rows, [&](auto s) { go(s, std::integral_constant<int, 2>{}); });
  return with_value_shape<false>(a.cols, a.rows, [&](auto s) { go(s, std::integral_constant<int, 1>{}); });
}

template <typename T, int kAct, bool kSym>
int launch(const QuantArgs& a, cudaStream_t st) {
  if (launch_rows<T, kAct>(a, st)) {
    LC_LAUNCH_CHECK();
    return LC_OK;
  }
  const int64_t cap = (int64_t)kNumSMsB200 * 8;
  launch_dependent(quant_any_kernel<T, kAct, kSym>, dim3((unsigned)(a.rows < cap ? a.rows : cap)), kThreads, 0, st, a);
  LC_LAUNCH_CHECK();
  return LC_OK;
}

template <typename T, int kAct>
int by_sym(const QuantArgs& a, cudaStream_t st) {
  return a.zeros ? launch<T, kAct, false>(a, st) : launch<T, kAct, true>(a, st);
}

template <typename T>
int by_act(const QuantArgs& a, int act, cudaStream_t st) {
  switch (act) {
    case kNone: return by_sym<T, kNone>(a, st);
    case kSilu: return by_sym<T, kSilu>(a, st);
    case kGelu: return by_sym<T, kGelu>(a, st);
    case kGeluTanh: return by_sym<T, kGeluTanh>(a, st);
    default: return LC_ERR_ARG;
  }
}

int quant_rows(const QuantArgs& a, int dtype, int act, cudaStream_t st) {
  switch (dtype) {
    case LC_F32: return by_act<float>(a, act, st);
    case LC_BF16: return by_act<__nv_bfloat16>(a, act, st);
    case LC_F16: return by_act<__half>(a, act, st);
    default: return LC_ERR_ARG;
  }
}

}  // namespace

int int8_quant_rows(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ldx, int8_t* codes, int64_t ldc,
                    float* scales, int32_t* zeros, cudaStream_t st) {
  return quant_rows(QuantArgs{x, x, rows, cols, ldx, ldx, ldc, codes, scales, zeros}, dtype, kNone, st);
}

}  // namespace lc

extern "C" LC_API int lc_int8_act_quant(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ldx, int8_t* codes,
                                        int64_t ldc, float* scales, int32_t* zeros, lc_stream_t stream) {
  using namespace lc;
  if (dtype < LC_F32 || dtype > LC_F16 || rows < 0 || cols <= 0 || ldx < 0 || ldc < cols) return LC_ERR_ARG;
  if (rows == 0) return LC_OK;
  if (!x || !codes || !scales) return LC_ERR_ARG;
  return int8_quant_rows(x, dtype, rows, cols, ldx, codes, ldc, scales, zeros, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" LC_API int lc_int8_gated_act_quant(const void* gate, const void* up, int dtype, int64_t rows, int64_t cols,
                                              int64_t ldg, int64_t ldu, int act, int8_t* codes, int64_t ldc,
                                              float* scales, int32_t* zeros, lc_stream_t stream) {
  using namespace lc;
  if (dtype < LC_F32 || dtype > LC_F16 || act < LC_ACT_SILU || act > LC_ACT_GELU_TANH) return LC_ERR_ARG;
  if (rows < 0 || cols <= 0 || ldg < 0 || ldu < 0 || ldc < cols) return LC_ERR_ARG;
  if (rows == 0) return LC_OK;
  if (!gate || !up || !codes || !scales) return LC_ERR_ARG;
  return quant_rows(QuantArgs{gate, up, rows, cols, ldg, ldu, ldc, codes, scales, zeros}, dtype, act,
                    reinterpret_cast<cudaStream_t>(stream));
}
