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
  begin_dependent();
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

// Rows that registers hold, by 16-byte vectors or, less aligned, by pairs or single values: x, the residual and the gate are
// read once, h and y written once; the weights come from the caches.  HBM-bound: 32768 x 4096 in bf16 with both norms and a gate
// takes 165 us, 6.5 TB/s or 99 % of a copy's rate.  A lane keeps its vectors as they lie in memory (x, then h) and unpacks
// them where it needs them: the registers of fp32 copies cost wide rows their occupancy (2048 x 16384 with two inputs: 84
// us, 51 this way).
template <typename T, int N, int kWarps, int kVecs, bool kCodes>
__global__ void __launch_bounds__(RowGroup<kWarps>::kThreads) norm_rows_kernel(NormArgs a) {
  using G = RowGroup<kWarps>;
  using P = Raw<T, N>;
  __shared__ float red[4 * kWarps];
  begin_dependent();
  const int64_t row = (int64_t)blockIdx.x * G::kRows + G::row();
  if (G::kRows > 1 && row >= a.rows) return;                           // a whole warp, and no barrier follows
  const int vecs = (int)(a.cols / N);
  const float inv_c = 1.f / (float)a.cols;
  const T* x = static_cast<const T*>(a.x) + row * a.ldx;
  const T* res = a.residual ? static_cast<const T*>(a.residual) + row * a.ldr : nullptr;
  const P* gate = a.gate ? reinterpret_cast<const P*>(static_cast<const T*>(a.gate) + row / a.rows_per_gate * a.cols) : nullptr;
  const P* pw = static_cast<const P*>(a.post_weight);
  const P* w = static_cast<const P*>(a.weight);
  P kept[kVecs], rr[kVecs];
#pragma unroll
  for (int k = 0; k < kVecs; ++k) {
    const int i = G::lane() + k * G::kLanes;
    kept[k] = i < vecs ? load_stream<T, N>(x + i * N) : pack<T, N>({});
    if (res) rr[k] = i < vecs ? load_stream<T, N>(res + i * N) : pack<T, N>({});
  }
  auto squares = [&](int k) {
    float v[N], s = 0.f;
    unpack<T, N>(kept[k], v);
#pragma unroll
    for (int j = 0; j < N; ++j) s = fmaf(v[j], v[j], s);
    return s;
  };
  if (a.h) {
    float post = 1.f;
    if (pw) {
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < kVecs; ++k) s += squares(k);
      post = rsqrtf(G::sum(s, red) * inv_c + a.eps);
    }
    P* h = reinterpret_cast<P*>(static_cast<T*>(a.h) + row * a.cols);
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      const int i = G::lane() + k * G::kLanes;
      if (i < vecs) {
        float v[N], f[N];
        unpack<T, N>(kept[k], v);
        if (pw) {
          unpack<T, N>(__ldg(pw + i), f);
#pragma unroll
          for (int j = 0; j < N; ++j) v[j] = v[j] * post * (f[j] + a.offset);
        }
        if (gate) {
          unpack<T, N>(__ldg(gate + i), f);
#pragma unroll
          for (int j = 0; j < N; ++j) v[j] *= f[j];
        }
        if (res) unpack<T, N>(rr[k], f);
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = res ? v[j] * a.scale + f[j] : v[j] * a.scale;
        kept[k] = pack<T, N>(v);
        h[i] = kept[k];
      }
    }
  }
  if (!w) return;
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < kVecs; ++k) s += squares(k);
  const float pre = rsqrtf(G::sum(s, red + kWarps) * inv_c + a.eps);
  auto normed = [&](int k, int i, float (&v)[N]) {
    float f[N];
    unpack<T, N>(kept[k], v);
    unpack<T, N>(__ldg(w + i), f);
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = v[j] * pre * (f[j] + a.offset);
  };
  if (!kCodes || a.y) {
    P* y = reinterpret_cast<P*>(static_cast<T*>(a.y) + row * a.cols);
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      const int i = G::lane() + k * G::kLanes;
      if (i < vecs) {
        float v[N];
        normed(k, i, v);
        y[i] = pack<T, N>(v);
      }
    }
  }
  if constexpr (kCodes) {
    // kept in fp32 from the range to the codes where registers hold them, else formed again (2048 x 4096 in bf16: 12.3 us,
    // 12.8 with all formed again; 19 x 4092 3.2 and 3.7)
    constexpr bool kHold = kVecs * N <= 32;
    const bool sym = a.zeros == nullptr;
    float mn = 0.f, mx = 0.f, held[kHold ? kVecs : 1][N];
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      const int i = G::lane() + k * G::kLanes;
      if (i < vecs) {
        float(&v)[N] = held[kHold ? k : 0];
        normed(k, i, v);
#pragma unroll
        for (int j = 0; j < N; ++j) mx = nan_max(mx, v[j]), mn = nan_min(mn, v[j]);
      }
    }
    G::range(mn, mx, red + 2 * kWarps);
    const RowQuant q = row_quant_of(mn, mx, sym);
    int8_t* out = a.codes + row * a.ldc;
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      const int i = G::lane() + k * G::kLanes;
      if (i < vecs) {
        float(&v)[N] = held[kHold ? k : 0];
        if (!kHold) normed(k, i, v);
        store_row_codes<N>(out + i * N, v, q, sym);
      }
    }
    if (G::lane() == 0) {
      a.scales[row] = q.s;
      if (!sym) a.zeros[row] = q.z;
    }
  }
}

// whether norm_rows_kernel took the rows
template <typename T>
bool launch_rows(const NormArgs& a, cudaStream_t st) {
  constexpr int N = Elem<T>::kPerVec;
  if (a.rows > 0x7fffffff) return false;
  // whether every row begins at a multiple of n values; NULL counts as one
  auto by = [&](int n) {
    bool fits = a.cols % n == 0 &&
                (a.rows == 1 || (a.ldx % n == 0 && (!a.residual || a.ldr % n == 0) && (!a.codes || a.ldc % n == 0))) &&
                reinterpret_cast<uintptr_t>(a.codes) % n == 0;
    for (const void* p : {a.x, a.residual, a.post_weight, a.gate, a.weight, (const void*)a.h, (const void*)a.y})
      fits = fits && reinterpret_cast<uintptr_t>(p) % (n * sizeof(T)) == 0;
    return fits;
  };
  auto go = [&](auto shape, auto width) {
    using S = decltype(shape);
    using G = RowGroup<S::kWarps>;
    const dim3 grid((unsigned)((a.rows + G::kRows - 1) / G::kRows));
    constexpr int kWidth = decltype(width)::value;
    if (a.codes) launch_dependent(norm_rows_kernel<T, kWidth, S::kWarps, S::kVecs, true>, grid, G::kThreads, 0, st, a);
    else launch_dependent(norm_rows_kernel<T, kWidth, S::kWarps, S::kVecs, false>, grid, G::kThreads, 0, st, a);
  };
  if (by(N)) return with_row_shape<true>(a.cols / N, a.rows, [&](auto s) { go(s, std::integral_constant<int, N>{}); });
  if (by(2)) return with_value_shape<true>(a.cols / 2, a.rows, [&](auto s) { go(s, std::integral_constant<int, 2>{}); });
  return with_value_shape<true>(a.cols, a.rows, [&](auto s) { go(s, std::integral_constant<int, 1>{}); });
}

template <typename T>
int launch(const NormArgs& a, cudaStream_t st) {
  if (launch_rows<T>(a, st)) {
    LC_LAUNCH_CHECK();
    return LC_OK;
  }
  const int64_t cap = (int64_t)kNumSMsB200 * 8;
  launch_dependent(norm_any_kernel<T>, dim3((unsigned)(a.rows < cap ? a.rows : cap)), kThreads, 0, st, a);
  LC_LAUNCH_CHECK();
  return LC_OK;
}

}  // namespace
}  // namespace lc

extern "C" LC_API int lc_residual_norm(const lc_residual_norm_args* args_host, lc_stream_t stream) {
  using namespace lc;
  if (!args_host) return LC_ERR_ARG;
  const lc_residual_norm_args& p = *args_host;
  if (p.dtype < LC_F32 || p.dtype > LC_F16 || p.rows < 0 || p.cols <= 0 || p.ldx < 0 || p.ldr < 0) return LC_ERR_ARG;
  if (p.gate && (p.gate_rows <= 0 || p.rows % p.gate_rows != 0)) return LC_ERR_SHAPE;
  if (p.rows == 0) return LC_OK;
  if (!p.x) return LC_ERR_ARG;
  // without h the norm is x's own: nothing may change x first
  if (!p.h && (p.residual || p.post_weight || p.gate || p.scale != 1.0 || !p.weight)) return LC_ERR_ARG;
  if ((p.weight != nullptr) != (p.y != nullptr || p.codes != nullptr)) return LC_ERR_ARG;
  if (p.codes && (!p.scales || p.ldc < p.cols)) return LC_ERR_ARG;
  NormArgs a{p.x, p.residual, p.post_weight, p.gate, p.weight, p.rows, p.cols, p.ldx, p.ldr,
             p.gate ? p.rows / p.gate_rows : p.rows, p.ldc, (float)p.scale, (float)p.eps, (float)p.weight_offset,
             p.h, p.y, p.codes, p.scales, p.zeros};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  switch (p.dtype) {
    case LC_F32: return launch<float>(a, st);
    case LC_BF16: return launch<__nv_bfloat16>(a, st);
    default: return launch<__half>(a, st);
  }
}
