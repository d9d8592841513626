// The residual add of a decoder block with the norms on both sides of it, for the block forms that the plain
// x + attn(norm(x)) does not cover (a norm after the sub-layer, a gate or layer scale on its output, a residual
// multiplier), optionally with the 8-bit quantisation that the next integer linear needs:
//
//   t = x                       or  x * rsqrt(mean(x^2) + eps) * (post_weight + offset)
//   h = residual + scale * gate * t                       rounded to the tensor type and kept
//   y = h * rsqrt(mean(h^2) + eps) * (weight + offset)    rounded once, or quantised from fp32 (row_quant.cuh)
//
// Everything between the loads and the two roundings is fp32.  y is formed from h as it is kept, so the stream of
// a model that stores h in 16 bits and one that re-reads it agree.
#include <type_traits>

#include "row_quant.cuh"

namespace lc {
namespace {

constexpr int kThreads = 256;

struct NormArgs {
  const void *x, *residual, *post_weight, *gate, *weight;
  int64_t rows, cols, ldx, ldr, rows_per_gate, ldc;
  float scale, eps, offset;
  void *h, *y;
  int8_t* codes;
  float* scales;
  int32_t* zeros;
};

__device__ __forceinline__ float block_sum(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = red[0];
#pragma unroll
  for (int w = 1; w < kThreads / 32; ++w) s += red[w];
  return s;
}

// Any width and alignment: a CTA per row; h goes to memory and is read back by the thread that wrote it.
template <typename T>
__global__ void __launch_bounds__(kThreads) norm_any_kernel(NormArgs a) {
  using E = Elem<T>;
  __shared__ float red[16];
  const float inv_c = 1.f / (float)a.cols;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    const T* h = a.h ? static_cast<const T*>(a.h) + row * a.cols : x;
    if (a.h) {
      T* hw = static_cast<T*>(a.h) + row * a.cols;
      const T* pw = static_cast<const T*>(a.post_weight);
      const T* gate = a.gate ? static_cast<const T*>(a.gate) + row / a.rows_per_gate * a.cols : nullptr;
      const T* res = a.residual ? static_cast<const T*>(a.residual) + row * a.ldr : nullptr;
      float post = 1.f;
      if (pw) {
        float s = 0.f;
        for (int64_t c = threadIdx.x; c < a.cols; c += kThreads) s += E::to_f(x[c]) * E::to_f(x[c]);
        post = rsqrtf(block_sum(s, red) * inv_c + a.eps);
      }
      for (int64_t c = threadIdx.x; c < a.cols; c += kThreads) {
        float t = E::to_f(x[c]);
        if (pw) t = t * post * (E::to_f(pw[c]) + a.offset);
        if (gate) t *= E::to_f(gate[c]);
        t *= a.scale;
        if (res) t += E::to_f(res[c]);
        hw[c] = E::from_f(t);
      }
    }
    if (!a.weight) continue;
    const T* w = static_cast<const T*>(a.weight);
    float s = 0.f;
    for (int64_t c = threadIdx.x; c < a.cols; c += kThreads) s += E::to_f(h[c]) * E::to_f(h[c]);
    const float pre = rsqrtf(block_sum(s, red) * inv_c + a.eps);
    auto value = [&](int64_t c) { return E::to_f(h[c]) * pre * (E::to_f(w[c]) + a.offset); };
    if (a.y) {
      T* y = static_cast<T*>(a.y) + row * a.cols;
      for (int64_t c = threadIdx.x; c < a.cols; c += kThreads) y[c] = E::from_f(value(c));
    }
    if (a.codes) {
      int8_t* out = a.codes + row * a.ldc;
      auto quantise = [&](auto sym_tag) {
        constexpr bool kSym = decltype(sym_tag)::value;
        RowRange<kSym> m;
        for (int64_t c = threadIdx.x; c < a.cols; c += kThreads) m.add(value(c));
        m.warp_reduce();
        __syncthreads();
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m.mx, red[8 + (threadIdx.x >> 5)] = m.mn;
        __syncthreads();
        float mx = red[0], mn = red[8];
#pragma unroll
        for (int i = 1; i < kThreads / 32; ++i) mx = nan_max(mx, red[i]), mn = nan_min(mn, red[8 + i]);
        const RowQuant q = row_quant<kSym>(mn, mx);
        for (int64_t c = threadIdx.x; c < a.cols; c += kThreads)
          out[c] = q.bad ? (int8_t)0 : (int8_t)row_code<kSym>(value(c), q);
        if (threadIdx.x == 0) {
          a.scales[row] = q.s;
          if (!kSym) a.zeros[row] = q.z;
        }
      };
      if (a.zeros) quantise(std::false_type{});
      else quantise(std::true_type{});
    }
  }
}

template <typename T>
int launch(const NormArgs& a, cudaStream_t st) {
  const int64_t cap = (int64_t)kNumSMsB200 * 8;
  norm_any_kernel<T><<<(unsigned)(a.rows < cap ? a.rows : cap), kThreads, 0, st>>>(a);
  LC_LAUNCH_CHECK();
  return LC_OK;
}

}  // namespace
}  // namespace lc

extern "C" LC_API int lc_residual_norm(const void* x, const void* residual, const void* post_weight, const void* gate,
                                       int64_t gate_rows, const void* weight, int dtype, int64_t rows, int64_t cols,
                                       int64_t ldx, int64_t ldr, float scale, float eps, float weight_offset, void* h,
                                       void* y, int8_t* codes, int64_t ldc, float* scales, int32_t* zeros,
                                       lc_stream_t stream) {
  using namespace lc;
  if (dtype < LC_F32 || dtype > LC_F16 || rows < 0 || cols <= 0 || ldx < 0 || ldr < 0) return LC_ERR_ARG;
  if (gate && (gate_rows <= 0 || rows % gate_rows != 0)) return LC_ERR_SHAPE;
  if (rows == 0) return LC_OK;
  if (!x) return LC_ERR_ARG;
  // without h the norm is x's own: nothing may change x first
  if (!h && (residual || post_weight || gate || scale != 1.f)) return LC_ERR_ARG;
  if (!h && !weight) return LC_ERR_ARG;
  if ((weight != nullptr) != (y != nullptr || codes != nullptr)) return LC_ERR_ARG;
  if (codes && (!scales || ldc < cols)) return LC_ERR_ARG;
  NormArgs a{x, residual, post_weight, gate, weight, rows, cols, ldx, ldr, gate ? rows / gate_rows : rows, ldc,
             scale, eps, weight_offset, h, y, codes, scales, zeros};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  switch (dtype) {
    case LC_F32: return launch<float>(a, st);
    case LC_BF16: return launch<__nv_bfloat16>(a, st);
    default: return launch<__half>(a, st);
  }
}
