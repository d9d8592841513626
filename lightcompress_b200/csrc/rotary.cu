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

constexpr int kThreads = 128;

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

// x / d for x < 2^20 and d <= 1024 as a multiplication: m = ceil(2^32 / d) is off by e < d / 2^32 of itself, and
// x * e < 2^30
struct Divider {
  uint32_t d, m;
};
__device__ __forceinline__ uint32_t quotient(uint32_t x, const Divider& v) { return v.d == 1 ? x : __umulhi(x, v.m); }

// W elements move as one access, as many as the alignment of q, k and of the halves allows.  A head is R/2/W pieces of two
// accesses that turn together (halves) or R/W pieces that turn by themselves (interleaved; R/2 pairs with W = 1), and
// (D - R)/W that are copied; an item is up to U pieces that lie `items` pieces apart, so that narrow accesses neither cost
// their index arithmetic each nor wait for one another (613 tokens of 20 heads of 192, of which 142 turn: 7.7 us, 9.1 with
// U = 1).  A CTA takes `per_cta` tokens, whose places, cosines and sines it forms in shared memory first.
//
// HBM-bound: q and k are read and written once.  What carries it is warps on the SM: 16 CTAs of 128 threads at 32 registers
// take 86.3 us for 16384 tokens of 64 heads of 128 in bf16 (6.2 TB/s, 95 % of a copy's rate); 34 registers and 256 threads
// took 102, two items a thread with their loads ahead of the angles (64 registers) 128.
template <typename T, int W> struct alignas(sizeof(T) * W) Pack { T v[W]; };

struct Shape {
  int turned, copied;        // pieces of a head
  int turned_items, per_head;
  int heads;                 // q's and k's
  int per_cta;               // tokens
  Divider by_head, by_token; // per_head; heads
};

template <typename T, int W, int U, bool kInter>
__global__ void __launch_bounds__(kThreads, U == 1 ? 16 : 10) rotary_kernel(RotaryArgs a, Shape sh) {
  using E = Elem<T>;
  using P = Pack<T, W>;
  extern __shared__ float2 cs[];
  begin_dependent();
  const int half = a.R / 2;
  const int64_t tok0 = (int64_t)blockIdx.x * sh.per_cta;
  const int tokens = (int)min((int64_t)sh.per_cta, a.B * a.T - tok0);
  int2* place = reinterpret_cast<int2*>(cs + sh.per_cta * half);         // (b, t) of each token
  for (int j = threadIdx.x; j < tokens; j += kThreads) {
    const int64_t tok = tok0 + j, b = a.B == 1 ? 0 : tok / a.T;
    place[j] = make_int2((int)b, (int)(tok - b * a.T));
  }
  __syncthreads();
  for (int j = threadIdx.x; j < tokens * half; j += kThreads) {
    const int tl = j / half;
    cs[j] = turn(a.positions[place[tl].x * a.pos_b + place[tl].y], a.inv_freq[j - tl * half], a.scale);
  }
  __syncthreads();
  const uint32_t items = (uint32_t)(tokens * sh.heads * sh.per_head);
#pragma unroll(U == 1 ? 2 : 1)
  for (uint32_t idx = blockIdx.y * kThreads + threadIdx.x; idx < items; idx += gridDim.y * kThreads) {
    const uint32_t th = quotient(idx, sh.by_head);
    int i = (int)(idx - th * sh.per_head);
    const uint32_t tl = quotient(th, sh.by_token);
    int head = (int)(th - tl * sh.heads);
    const int2 at = place[tl];
    const bool is_k = head >= a.q.heads;
    const Heads& s = is_k ? a.k : a.q;
    if (is_k) head -= a.q.heads;
    const T* in = static_cast<const T*>(s.in) + at.x * s.in_b + at.y * s.in_t + head * s.in_h;
    T* out = static_cast<T*>(s.out) + at.x * s.out_b + at.y * s.out_t + head * s.out_h;
    const float2* w = cs + tl * half;
    if (i < sh.turned_items) {
      constexpr int kStep = kInter && W == 1 ? 2 : W;        // elements from piece to piece
      P x1[U], x2[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int e = (i + u * sh.turned_items) * kStep;
        if (U == 1 || i + u * sh.turned_items < sh.turned) {
          x1[u] = *reinterpret_cast<const P*>(in + e);
          if (!kInter) x2[u] = *reinterpret_cast<const P*>(in + half + e);
          else if (W == 1) x2[u] = *reinterpret_cast<const P*>(in + e + 1);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int e = (i + u * sh.turned_items) * kStep;
        if (U > 1 && i + u * sh.turned_items >= sh.turned) continue;
        if constexpr (kInter && W > 1) {
#pragma unroll
          for (int j = 0; j < W; j += 2) {
            const float2 c = w[(e + j) / 2];
            const float p = E::to_f(x1[u].v[j]), q = E::to_f(x1[u].v[j + 1]);
            x1[u].v[j] = E::from_f(p * c.x - q * c.y);
            x1[u].v[j + 1] = E::from_f(q * c.x + p * c.y);
          }
          *reinterpret_cast<P*>(out + e) = x1[u];
        } else {
#pragma unroll
          for (int j = 0; j < W; ++j) {
            const float2 c = w[kInter ? e / 2 : e + j];
            const float p = E::to_f(x1[u].v[j]), q = E::to_f(x2[u].v[j]);
            x1[u].v[j] = E::from_f(p * c.x - q * c.y);
            x2[u].v[j] = E::from_f(q * c.x + p * c.y);
          }
          *reinterpret_cast<P*>(out + e) = x1[u];
          *reinterpret_cast<P*>(out + (kInter ? 1 : half) + e) = x2[u];
        }
      }
    } else {
      i -= sh.turned_items;
      const int step = sh.per_head - sh.turned_items;
      P x[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (U == 1 || i + u * step < sh.copied) x[u] = *reinterpret_cast<const P*>(in + a.R + (i + u * step) * W);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (U == 1 || i + u * step < sh.copied) *reinterpret_cast<P*>(out + a.R + (i + u * step) * W) = x[u];
    }
  }
}

template <typename T, int W, bool kInter>
int launch_packed(const RotaryArgs& a, cudaStream_t st) {
  constexpr int kFull = Elem<T>::kPerVec / W, U = kFull < 4 ? kFull : 4;
  Shape sh;
  sh.turned = kInter && W > 1 ? a.R / W : a.R / 2 / W;
  sh.copied = (a.D - a.R) / W;
  sh.turned_items = (sh.turned + U - 1) / U;
  sh.per_head = sh.turned_items + (sh.copied + U - 1) / U;
  sh.heads = a.q.heads + a.k.heads;
  const int per_token = sh.heads * sh.per_head;
  if (sh.per_head > 1024 || per_token >= 1 << 20) return LC_ERR_SHAPE;
  // two items a thread at least, so that a token of few heads does not leave a CTA idle; at most 16 KB of angles
  sh.per_cta = per_token >= 2 * kThreads ? 1 : (2 * kThreads + per_token - 1) / per_token;
  const int room = 2048 / (a.R / 2) > 0 ? 2048 / (a.R / 2) : 1;
  if (sh.per_cta > room) sh.per_cta = room;
  // a few tokens: one to a CTA, or their items spread over several CTAs, each of which forms the angles -- up to the CTAs
  // that run at once, so that the chain of angles and items is short (in a graph, of which 2.2 are a launch: 24 tokens of 2
  // heads of 192 2.4 us, 5.8 with all in two CTAs; 613 tokens of 20 heads of 192, 142 of them turned, 9.1 us with single
  // accesses an item, 13.6 with a quarter of the CTAs)
  constexpr int64_t kAtOnce = 16 * kNumSMsB200;
  const int64_t tokens = a.B * a.T, spread = (tokens + kAtOnce - 1) / kAtOnce;
  if (sh.per_cta > spread) sh.per_cta = (int)spread;
  auto divider = [](int d) { return Divider{(uint32_t)d, (uint32_t)(((1ull << 32) + d - 1) / d)}; };
  sh.by_head = divider(sh.per_head);
  sh.by_token = divider(sh.heads);
  const int64_t grid = (tokens + sh.per_cta - 1) / sh.per_cta;
  if (grid > 0x7fffffff) return LC_ERR_SHAPE;
  int64_t parts = (kAtOnce + grid - 1) / grid;
  const int64_t most = ((int64_t)sh.per_cta * per_token + kThreads - 1) / kThreads;
  if (parts > most) parts = most;
  LC_CHECK_CUDA(launch_dependent(rotary_kernel<T, W, U, kInter>, dim3((unsigned)grid, (unsigned)parts), kThreads,
                                 (size_t)sh.per_cta * (a.R / 2 * sizeof(float2) + sizeof(int2)), st, a, sh));
  LC_LAUNCH_CHECK();
  return LC_OK;
}

// whether every vector of V elements that the kernel touches is aligned to its size
template <typename T>
bool fits(const RotaryArgs& a, int v, bool inter) {
  if (a.D % v || a.R % v || (!inter && a.R / 2 % v)) return false;
  for (const Heads* h : {&a.q, &a.k}) {
    if (h->heads == 0) continue;
    const uintptr_t bytes = sizeof(T) * v;
    if (reinterpret_cast<uintptr_t>(h->in) % bytes || reinterpret_cast<uintptr_t>(h->out) % bytes) return false;
    for (int64_t s : {h->in_b, h->in_t, h->in_h, h->out_b, h->out_t, h->out_h})
      if (s % v) return false;
  }
  return true;
}

template <typename T, bool kInter>
int by_width(const RotaryArgs& a, cudaStream_t st) {
  constexpr int N = Elem<T>::kPerVec;
  if (fits<T>(a, N, kInter)) return launch_packed<T, N, kInter>(a, st);
  if (N > 4 && fits<T>(a, 4, kInter)) return launch_packed<T, 4, kInter>(a, st);
  if (fits<T>(a, 2, kInter)) return launch_packed<T, 2, kInter>(a, st);
  return launch_packed<T, 1, kInter>(a, st);
}

template <typename T>
int launch(const RotaryArgs& a, int interleaved, cudaStream_t st) {
  return interleaved ? by_width<T, true>(a, st) : by_width<T, false>(a, st);
}

}  // namespace
}  // namespace lc

extern "C" LC_API int lc_rotary_embed(const lc_rotary_embed_args* args_host, lc_stream_t stream) {
  using namespace lc;
  if (!args_host) return LC_ERR_ARG;
  const lc_rotary_embed_args& p = *args_host;
  if (p.dtype < LC_F32 || p.dtype > LC_F16 || p.batch < 0 || p.tokens < 0 || p.q_heads < 0 || p.k_heads < 0) return LC_ERR_ARG;
  if (p.head_dim <= 0 || p.rotary_dim <= 0) return LC_ERR_ARG;
  if (p.rotary_dim % 2 != 0 || p.rotary_dim > p.head_dim || p.head_dim > 1024) return LC_ERR_SHAPE;
  if (p.q_heads > 1023 || p.k_heads > 1023 || p.q_heads + p.k_heads > 1023) return LC_ERR_SHAPE;
  if (p.batch > (1 << 30) || p.tokens > (1 << 30)) return LC_ERR_SHAPE;
  if (p.batch == 0 || p.tokens == 0 || p.q_heads + p.k_heads == 0) return LC_OK;
  if (!p.positions || !p.inv_freq || (p.q_heads && (!p.q || !p.q_out)) || (p.k_heads && (!p.k || !p.k_out))) return LC_ERR_ARG;
  // outputs lie as (batch, tokens, heads, head_dim) without gaps, unless they are the inputs themselves
  auto heads = [&](const void* in, void* out, int64_t n, int64_t sb, int64_t st, int64_t sh) {
    const int64_t row = n * p.head_dim;
    return in == out ? Heads{in, out, (int)n, sb, st, sh, sb, st, sh}
                     : Heads{in, out, (int)n, sb, st, sh, row * p.tokens, row, p.head_dim};
  };
  RotaryArgs a{heads(p.q, p.q_out, p.q_heads, p.q_b, p.q_t, p.q_h), heads(p.k, p.k_out, p.k_heads, p.k_b, p.k_t, p.k_h),
               p.positions, p.pos_b, p.inv_freq, p.batch, p.tokens, (int)p.head_dim, (int)p.rotary_dim, (float)p.scale};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int interleaved = p.interleaved != 0;
  switch (p.dtype) {
    case LC_F32: return launch<float>(a, interleaved, st);
    case LC_BF16: return launch<__nv_bfloat16>(a, interleaved, st);
    default: return launch<__half>(a, interleaved, st);
  }
}
