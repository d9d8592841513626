// Rotary embedding of q and k from positions: for pair i of the first R of D elements of a head,
//   angle = position * inv_freq[i],  (x1, x2) -> scale * (x1 cos - x2 sin, x2 cos + x1 sin)
// with pairs (i, i + R/2) or, interleaved, (2i, 2i + 1); the other D - R elements are copied.  inv_freq carries
// whatever scaling for long contexts the model asks for.
//
// The angle of a far position needs more than 32 bits: position * inv_freq is formed in fp64 (exact: 31 + 24 bits
// would need 55, the rounding of the 53rd is below 1e-7 of a turn for positions under 2^31), taken modulo 2 pi
// there, and sine and cosine of the remainder in [-pi, pi] are fp32.  They are computed once per token and pair
// and serve all heads of q and k.
#include "lc_common.cuh"

namespace lc {
namespace {

constexpr int kThreads = 256;

struct Heads {
  const void* in;
  void* out;
  int heads;
  int64_t in_b, in_t, in_h, out_b, out_t, out_h;
};

struct RotaryArgs {
  Heads q, k;
  const int64_t* positions;
  int64_t pos_b;
  const float* inv_freq;
  int64_t B, T;
  int D, R;
  float scale;
};

__device__ __forceinline__ float2 turn(int64_t pos, float freq, float scale) {
  const double angle = (double)pos * (double)freq;
  const double n = rint(angle * 0.15915494309189535);                 // 1 / (2 pi)
  // 2 pi = hi + lo: n * hi is subtracted exactly (fma), lo carries the rest
  const double r = fma(-n, 2.4492935982947064e-16, fma(-n, 6.283185307179586, angle));
  float s, c;
  sincosf((float)r, &s, &c);
  return make_float2(c * scale, s * scale);
}

// One CTA per token: the token's cosines and sines go to shared memory, then every head of q and k is turned.
template <typename T, bool kInter>
__global__ void __launch_bounds__(kThreads) rotary_any_kernel(RotaryArgs a) {
  using E = Elem<T>;
  extern __shared__ float2 cs[];
  const int half = a.R / 2;
  for (int64_t tok = blockIdx.x; tok < a.B * a.T; tok += gridDim.x) {
    const int64_t b = tok / a.T, t = tok % a.T;
    __syncthreads();
    for (int i = threadIdx.x; i < half; i += kThreads)
      cs[i] = turn(a.positions[b * a.pos_b + t], a.inv_freq[i], a.scale);
    __syncthreads();
    const int per_head = half + (a.D - a.R);          // a pair, or an element that is copied
    for (int idx = threadIdx.x; idx < (a.q.heads + a.k.heads) * per_head; idx += kThreads) {
      int head = idx / per_head;
      const int i = idx % per_head;
      const bool is_k = head >= a.q.heads;
      const Heads& s = is_k ? a.k : a.q;
      if (is_k) head -= a.q.heads;
      const T* in = static_cast<const T*>(s.in) + b * s.in_b + t * s.in_t + head * s.in_h;
      T* out = static_cast<T*>(s.out) + b * s.out_b + t * s.out_t + head * s.out_h;
      if (i < half) {
        const int i1 = kInter ? 2 * i : i, i2 = kInter ? 2 * i + 1 : i + half;
        const float x1 = E::to_f(in[i1]), x2 = E::to_f(in[i2]);
        const float2 w = cs[i];
        out[i1] = E::from_f(x1 * w.x - x2 * w.y);
        out[i2] = E::from_f(x2 * w.x + x1 * w.y);
      } else {
        out[a.R + i - half] = in[a.R + i - half];
      }
    }
  }
}

template <typename T>
int launch(const RotaryArgs& a, int interleaved, cudaStream_t st) {
  const int64_t tokens = a.B * a.T, cap = (int64_t)kNumSMsB200 * 8;
  const unsigned grid = (unsigned)(tokens < cap ? tokens : cap);
  const size_t smem = (size_t)a.R / 2 * sizeof(float2);
  if (interleaved) rotary_any_kernel<T, true><<<grid, kThreads, smem, st>>>(a);
  else rotary_any_kernel<T, false><<<grid, kThreads, smem, st>>>(a);
  LC_LAUNCH_CHECK();
  return LC_OK;
}

}  // namespace
}  // namespace lc

extern "C" LC_API int lc_rotary_embed(const void* q, void* q_out, int q_heads, int64_t q_b, int64_t q_t, int64_t q_h,
                                      const void* k, void* k_out, int k_heads, int64_t k_b, int64_t k_t, int64_t k_h,
                                      const int64_t* positions, int64_t pos_b, const float* inv_freq, int dtype,
                                      int64_t batch, int64_t tokens, int head_dim, int rotary_dim, int interleaved,
                                      float scale, lc_stream_t stream) {
  using namespace lc;
  if (dtype < LC_F32 || dtype > LC_F16 || batch < 0 || tokens < 0 || q_heads < 0 || k_heads < 0) return LC_ERR_ARG;
  if (head_dim <= 0 || rotary_dim <= 0) return LC_ERR_ARG;
  if (rotary_dim % 2 != 0 || rotary_dim > head_dim || head_dim > 1024 || q_heads > 65536 || k_heads > 65536)
    return LC_ERR_SHAPE;
  if (batch > (1 << 30) || tokens > (1 << 30)) return LC_ERR_SHAPE;
  if (batch == 0 || tokens == 0 || q_heads + k_heads == 0) return LC_OK;
  if (!positions || !inv_freq || (q_heads && (!q || !q_out)) || (k_heads && (!k || !k_out))) return LC_ERR_ARG;
  // outputs lie as (batch, tokens, heads, head_dim) without gaps, unless they are the inputs themselves
  auto heads = [&](const void* in, void* out, int n, int64_t sb, int64_t st, int64_t sh) {
    const int64_t row = (int64_t)n * head_dim;
    return in == out ? Heads{in, out, n, sb, st, sh, sb, st, sh}
                     : Heads{in, out, n, sb, st, sh, row * tokens, row, head_dim};
  };
  RotaryArgs a{heads(q, q_out, q_heads, q_b, q_t, q_h), heads(k, k_out, k_heads, k_b, k_t, k_h), positions, pos_b,
               inv_freq, batch, tokens, head_dim, rotary_dim, scale};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  switch (dtype) {
    case LC_F32: return launch<float>(a, interleaved, st);
    case LC_BF16: return launch<__nv_bfloat16>(a, interleaved, st);
    default: return launch<__half>(a, interleaved, st);
  }
}
