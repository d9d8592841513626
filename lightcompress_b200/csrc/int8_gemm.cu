// 8-bit integer linear: C[m][n] = (sum_k (A[m][k] - a_z[m]) B[n][k]) * a_s[m] * b_s[n] (+ bias[n]), A (M x K) int8
// codes of the activations with a scale (and zero point) per token, B (N x K) int8 weights with a scale per
// output channel: the product behind the reference's VllmQuantLinearInt8
// (llmc/compression/quantization/module_utils.py:145-209).
//
// The sum of products is a whole number held exactly in 32 bits, so its value depends neither on the tile nor on
// how the contraction is split; the zero point enters as -a_z[m] * b_sum[n] in the same 32-bit arithmetic (the
// bounds on K keep the final sum inside 32 bits; what wraps on the way wraps back).  After that there are two
// fp32 multiplications and an addition, in this order, and one rounding to the output type.
#include "row_quant.cuh"
#include "umma_common.cuh"

namespace lc {

int int8_quant_rows(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ldx, int8_t* codes, int64_t ldc,
                    float* scales, int32_t* zeros, cudaStream_t st);

namespace {

using namespace umma;

struct Int8Args {
  const void* x;           // a token that the kernel quantises itself (then a, a_s and a_z are not read)
  int sym, wide;           // wide: x is 16-byte aligned
  const int8_t* a;
  const int8_t* b;
  const float* a_s;
  const int32_t* a_z;      // NULL: no zero points
  const float* b_s;
  const int32_t* b_sum;
  const void* bias;        // out_dtype, or NULL
  void* c;                 // [M][N]
  int32_t* status;
  int64_t lda, ldb;
  int M, N, K;
};

// one element of the output; acc is the sum of the products of the codes
__device__ __forceinline__ float finish(int acc, float a_s, int a_z, float b_s, int b_sum, float bias) {
  const int whole = (int)((unsigned)acc - (unsigned)a_z * (unsigned)b_sum);
  return __fadd_rn(__fmul_rn(__fmul_rn(__int2float_rn(whole), a_s), b_s), bias);
}

// What a thread knows of its output channel.
struct Channel {
  float b_s, bias;
  int b_sum;
  bool ok;                 // the channel exists
};
template <typename T>
__device__ __forceinline__ Channel load_channel(const Int8Args& g, int n) {
  Channel c{0.f, 0.f, 0, n < g.N};
  if (c.ok) {
    c.b_s = g.b_s[n];
    if (g.bias) c.bias = Elem<T>::to_f(static_cast<const T*>(g.bias)[n]);
    if (g.b_sum) c.b_sum = g.b_sum[n];
  }
  return c;
}

// The outputs of C tokens of one channel.  s, z: the tokens' scales and zero points in shared memory (s 16-byte
// aligned); out: the first token's element, tokens N elements apart; count: how many of the C tokens exist.  All values
// are formed before the first store: stores may alias anything and would otherwise keep the loads behind them waiting
// (512 x 512 x 512 on pairs: 15.1 us with the loads between the stores, 7.8 this way).
template <typename T, int C>
__device__ __forceinline__ void finish_tokens(const uint32_t (&v)[C], const float* s, const int* z, bool zeros,
                                              const Channel& c, T* out, int64_t N, int count, bool lost) {
  float y[C];
#pragma unroll
  for (int i = 0; i < C; i += 4) {
    const float4 f = *reinterpret_cast<const float4*>(s + i);
    const int4 w = zeros ? *reinterpret_cast<const int4*>(z + i) : make_int4(0, 0, 0, 0);
    y[i] = finish((int)v[i], f.x, w.x, c.b_s, c.b_sum, c.bias);
    y[i + 1] = finish((int)v[i + 1], f.y, w.y, c.b_s, c.b_sum, c.bias);
    y[i + 2] = finish((int)v[i + 2], f.z, w.z, c.b_s, c.b_sum, c.bias);
    y[i + 3] = finish((int)v[i + 3], f.w, w.w, c.b_s, c.b_sum, c.bias);
  }
  if (lost) {
#pragma unroll
    for (int i = 0; i < C; ++i) y[i] = __int_as_float(0x7fffffff);
  }
  if (!c.ok) return;
  if (count >= C) {
#pragma unroll
    for (int i = 0; i < C; ++i) out[i * N] = Elem<T>::from_f(y[i]);
  } else {
#pragma unroll
    for (int i = 0; i < C; ++i)
      if (i < count) out[i * N] = Elem<T>::from_f(y[i]);
  }
}

// ---- weights as the 128-row operand, tokens as the columns ---------------------------------------------------
// One CTA per 128 output channels x NT tokens x one part of K (tcgen05 kind::i8, cta_group::1): the accumulator holds
// a channel per TMEM lane and a token per column, so a warp's store of one token is 32 neighbouring channels.  Both
// operands are K-major: a 128-byte swizzled row of a stage is 128 consecutive codes of one channel or token; K's ragged
// end and the rows behind the last are filled with zeros by the copy.
//
// Few tokens leave the weights as the only traffic that matters (N * K bytes), and N / 128 CTAs are too few to draw
// the HBM's bandwidth: K is split over the CTAs of a cluster.  Each CTA owns a run of the tile's tokens; every CTA lays its
// partial sums out by token in shared memory, one bulk copy takes an owner's run there, and the owner adds and finishes
// it (128 x 512 x 512 split in four: 8.3 us; 10.0 with stores of 4 bytes to the other CTAs).
//
// Both kernels, and the quantisations, norms and rotary embeddings around them, are launched as dependents of the kernel
// before them and wait for its end before they read anything, so that launching and setting up overlap (quantisation and
// product of 2 x 4096 x 4096: 9.2 us, 10.9 without).  Behind any other kernel, copy or fill the wait is over at once.
//
// What bounds it: for a few tokens the way of the weights from HBM, and 4 us of launch, first copies and exchange
// (1 x 4096 x 4096: 7.9 us with its quantisation, of which the weights' bytes are 2.6); for more, a k block's way from L2
// through a CTA's stages, 0.2 us.
constexpr int kRows = 128, kBlockK = 128, kStreamThreads = 256;
constexpr int kWeightBytes = kRows * kBlockK;
constexpr int kSmemMost = 227 * 1024;

// Bounded wait, asleep in the hardware between looks (up to 20 us each) instead of spinning: at the power limit that is
// 1.5 % of a large product.  False if a second has passed or another role has given up.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  auto look = [&] {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}"
        : "=r"(ok)
        : "r"(bar), "r"(parity), "r"(20000u)
        : "memory");
    return ok != 0;
  };
  if (look()) return true;
  uint64_t begin, now;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(begin));
  do {
    if (look()) return true;
    if (*abort_flag) return false;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
  } while (now - begin < 1000000000ull);
  *abort_flag = 1;
  return false;
}
// The same for a whole converged warp, with one answer for all of its lanes: each lane reads the clock and the flag for
// itself, and lanes that went separate ways would wait for one another at the next instruction that wants the whole warp.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, bar_wait(bar, parity, abort_flag));
}

// Called by every thread behind a barrier of the CTA: a wait that any thread of it gave up is reported, also where the
// thread that reports found what it waited for itself.
__device__ __forceinline__ void report_lost(int32_t* status, volatile int* abort_flag) {
  if (threadIdx.x == 0 && *abort_flag && status) atomicExch(status, (int)LC_ERR_TIMEOUT);
}

// kind::i8: D s32, A and B s8, both K-major
__host__ __device__ constexpr uint32_t idesc_i8(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

__device__ __forceinline__ void umma_i8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}"
      ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(acc)
      : "memory");
}

template <int C>
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&r)[C]) {
  static_assert(C == 8 || C == 16, "");
  if constexpr (C == 8)
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr)
                 : "memory");
  else
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
  tmem_wait_ld();
}

// true in one lane of a converged warp
__device__ __forceinline__ bool elect_one() {
  uint32_t is;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(is));
  return is != 0;
}

// Only once this CTA has its tensor memory: a product further on could otherwise take the columns that this one still
// needs, and wait for its end.
__device__ __forceinline__ void let_next_begin() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void grid_dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t in_cta(uint32_t addr, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
  return a;
}
// shared memory of this CTA -> that of a CTA of its cluster (dst and bar are addresses there)
__device__ __forceinline__ void copy_to_cta(uint32_t dst, uint32_t src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(dst), "r"(src), "r"(bytes), "r"(bar)
               : "memory");
}

struct Maps {
  CUtensorMap w, x;
};

// A single token is quantised by the product itself (kQuant): every CTA reads all of it for the range, before it asks for
// its weights (behind them a load took up to 2.5 us to come), keeps it in registers and lays the codes of its own part
// of K out as the copies would, while its first weights are on their way.  That saves a launch and a scratch buffer
// (4096 channels: 8.2 us, 9.0 in two launches; 11008 channels 11.2, 11.75); for more values than one a thread's 16 the
// separate kernel, which the product overlaps, is faster.
//
// Shared memory of a CTA: stages, barriers, the tokens' scales and zero points.  The CTA's own partial sums take the
// stages' place once its products are formed; those of the others land behind everything else where they are small, else
// behind its own (no CTA of the cluster may have products to form any more then).
constexpr int kRangeBytes = 2 * (kStreamThreads / 32) * 4;
template <int NT, bool kQuant> struct StreamSmem {
  static constexpr int kStage = kWeightBytes + (kQuant ? 0 : NT * kBlockK);
  static constexpr int kParts = (NT + 7) * kRows * 4;
  static constexpr bool kLandApart = NT <= 32;
  // stages that the partial sums need
  static constexpr int kLeast = ((kLandApart ? 1 : 2) * kParts + kStage - 1) / kStage;
  // codes: k blocks of codes that the CTA lays out itself
  __host__ __device__ static int codes(int stages) { return stages * kStage; }
  __host__ __device__ static int bars(int stages, int count) { return codes(stages) + (kQuant ? count * NT * kBlockK : 0); }
  __host__ __device__ static int scales(int stages, int count) {
    return bars(stages, count) + (8 * (2 * stages + 2) + 8 + 15) / 16 * 16;
  }
  __host__ __device__ static int ranges(int stages, int count) { return scales(stages, count) + NT * 8; }
  __host__ __device__ static int landing(int stages, int count) {
    return kLandApart ? ranges(stages, count) + (kQuant ? kRangeBytes : 0) : kParts;
  }
  __host__ __device__ static int bytes(int stages, int count, bool split) {
    return 1024 + ranges(stages, count) + (kQuant ? kRangeBytes : 0) + (kLandApart && split ? kParts : 0);
  }
};

// 16 neighbouring values of the token, as they lie in memory: chunk threadIdx.x of it
constexpr int kMostToken = kStreamThreads * 16;
template <typename T> struct Values {
  uint4 raw[sizeof(T)];
};

template <typename T>
__device__ __forceinline__ Values<T> load_token(const Int8Args& g) {
  Values<T> v;
  const int k = (int)threadIdx.x * 16;
  const T* x = static_cast<const T*>(g.x) + k;
  if (g.wide && k + 16 <= g.K) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T); ++i) v.raw[i] = reinterpret_cast<const uint4*>(x)[i];
  } else {
    T* p = reinterpret_cast<T*>(v.raw);
#pragma unroll
    for (int i = 0; i < 16; ++i) p[i] = k + i < g.K ? x[i] : Elem<T>::from_f(0.f);
  }
  return v;
}

// The token's scale and zero point, and its codes in k blocks [kb0, kb0 + count) as row 0 of their atoms.
template <typename T>
__device__ __forceinline__ void quantise_token(const Int8Args& g, const Values<T>& values, int kb0, int count, uint8_t* codes,
                                               int block_bytes, float* s_scale, int* s_zero, float* range) {
  float v[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = Elem<T>::to_f(reinterpret_cast<const T*>(values.raw)[i]);
  float mn = 0.f, mx = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) mn = nan_min(mn, v[i]), mx = nan_max(mx, v[i]);
  RowGroup<kStreamThreads / 32>::range(mn, mx, range);
  const RowQuant q = row_quant_of(mn, mx, g.sym);
  if (threadIdx.x == 0) {
    *s_scale = q.s;
    *s_zero = q.z;
  }
  const int kb = ((int)threadIdx.x >> 3) - kb0;
  if (kb >= 0 && kb < count) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float u[4] = {v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]};
      store_row_codes<4>(reinterpret_cast<int8_t*>(w + i), u, q, g.sym);
    }
    *reinterpret_cast<uint4*>(codes + kb * block_bytes + ((threadIdx.x & 7) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

template <typename T, int NT, bool kQuant>
__global__ void __launch_bounds__(kStreamThreads) stream_kernel(const __grid_constant__ Maps maps, Int8Args g, int splits,
                                                                int stages) {
  using Smem = StreamSmem<NT, kQuant>;
  constexpr int kStage = Smem::kStage;
  constexpr int kCols = NT < 32 ? 32 : NT;                 // tensor memory is allocated in powers of two from 32 columns
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
  const int blocks = (g.K + kBlockK - 1) / kBlockK, most = (blocks + splits - 1) / splits;
  const uint32_t bar0 = base + Smem::bars(stages, most);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(gen + Smem::bars(stages, most) + 8 * (2 * stages + 2));
  float* s_scale = reinterpret_cast<float*>(gen + Smem::scales(stages, most));
  int* s_zero = reinterpret_cast<int*>(s_scale + NT);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (stages + s); };
  const uint32_t acc_bar = bar0 + 8u * (2 * stages), land_bar = acc_bar + 8u;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x % splits;
  const int n0 = (int)(blockIdx.x / splits) * kRows, m0 = (int)blockIdx.y * NT;
  const int kb0 = (int)((int64_t)blocks * rank / splits), kb1 = (int)((int64_t)blocks * (rank + 1) / splits);
  const int count = kb1 - kb0;                             // at least 1: splits <= blocks
  const int tokens = min(NT, g.M - m0);
  // with splits: tokens [first, first + mine) of the tile are this CTA's to finish
  const int run = (tokens + splits - 1) / splits, first = rank * run, mine = max(0, min(run, tokens - first));

  Values<T> token;
  if constexpr (kQuant) {
    grid_dependency_wait();
    token = load_token<T>(g);
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    mbar_init(acc_bar, 1);
    mbar_init(land_bar, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if (splits > 1 && mine > 0) mbar_expect_tx(land_bar, (uint32_t)((splits - 1) * mine * kRows * 4));
    grid_dependency_wait();
    for (int i = 0; i < stages && i < count; ++i) {
      mbar_expect_tx(full_bar(i), kStage);
      tma_load_2d(base + i * kStage, &maps.w, (kb0 + i) * kBlockK, n0, full_bar(i));
    }
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"((uint32_t)kCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = *tmem_slot;
  let_next_begin();
  if (splits > 1) cluster_arrive();                        // waited for before anything is sent to another CTA
  const int group = warp >> 2;                             // of the two that share a channel
  const int c = (warp & 3) * 32 + lane, n = n0 + c;
  grid_dependency_wait();
  const Channel ch = load_channel<T>(g, n);
  const bool zeros = kQuant ? !g.sym : g.a_z != nullptr;
  if constexpr (kQuant) {
    quantise_token<T>(g, token, kb0, count, gen + Smem::codes(stages), NT * kBlockK, s_scale, s_zero,
                   reinterpret_cast<float*>(gen + Smem::ranges(stages, most)));
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");         // the MMAs read what was just written
    __syncthreads();
  } else {
    for (int t = (int)threadIdx.x - 64; t >= 0 && t < NT; t += kStreamThreads - 64) {
      s_scale[t] = t < tokens ? g.a_s[m0 + t] : 0.f;
      s_zero[t] = t < tokens && g.a_z ? g.a_z[m0 + t] : 0;
    }
  }

  int issued = 0;                                          // k blocks requested, known to thread 0
  if (warp == 0) {
    if (lane == 0) {
      if (!kQuant)
        for (int i = 0; i < stages && i < count; ++i)
          tma_load_2d(base + i * kStage + kWeightBytes, &maps.x, (kb0 + i) * kBlockK, m0, full_bar(i));
      int s = 0;
      uint32_t ph = 0;
      issued = min(stages, count);
      for (int i = stages; i < count; ++i) {
        if (!bar_wait(empty_bar(s), ph, abort_flag)) break;
        mbar_expect_tx(full_bar(s), kStage);
        tma_load_2d(base + s * kStage, &maps.w, (kb0 + i) * kBlockK, n0, full_bar(s));
        if (!kQuant) tma_load_2d(base + s * kStage + kWeightBytes, &maps.x, (kb0 + i) * kBlockK, m0, full_bar(s));
        issued = i + 1;
        if (++s == stages) s = 0, ph ^= 1u;
      }
    }
  } else if (warp == 1) {
    // The whole warp walks the stages and one lane issues, so that descriptors are formed in uniform registers; in a loop
    // of one lane alone they are moved there for every MMA, and the issue bound the kernel (64 x 128 tiles, 86 blocks: 0.28
    // us a block and 28.4 us in all; 0.20 and 22.4 this way; the pairs below gained 8 %).
    int s = 0;
    uint32_t ph = 0;
    const uint64_t dw0 = make_desc_mn_sw128(base, 16, 1024);
    const uint64_t dx0 = make_desc_mn_sw128(base + (kQuant ? Smem::codes(stages) : kWeightBytes), 16, 1024);
    for (int i = 0; i < count; ++i) {
      if (!warp_wait(full_bar(s), ph, abort_flag)) break;
      tcgen05_fence_after();
      const uint64_t at = (uint64_t)(s * (kStage >> 4)), xat = kQuant ? (uint64_t)(i * (NT * kBlockK >> 4)) : at;
      if (elect_one()) {
#pragma unroll
        for (int j = 0; j < kBlockK / 32; ++j)
          umma_i8(tmem, dw0 + at + j * 2, dx0 + xat + j * 2, idesc_i8(kRows, NT), (i | j) ? 1u : 0u);
        umma_commit(empty_bar(s));
      }
      __syncwarp();
      if (++s == stages) s = 0, ph ^= 1u;
    }
    if (elect_one()) umma_commit(acc_bar);                 // arrives once the MMAs issued so far have retired
  }
  __syncwarp();
  // the accumulator (or, after an expired wait, the retirement of what was issued)
  if (!bar_wait(acc_bar, 0, abort_flag))
    for (uint32_t it = 0; it < kSpinLimit && !mbar_test(acc_bar, 0); ++it) __nanosleep(50);
  __syncwarp();
  tcgen05_fence_after();
  __syncthreads();
  bool ok = *abort_flag == 0;
  if (!ok) {
    // the copies still in flight land before the CTA's shared memory is used again or released
    if (threadIdx.x == 0)
      for (int i = issued > stages ? issued - stages : 0; i < issued; ++i)
        for (uint32_t it = 0; it < kSpinLimit && !mbar_test(full_bar(i % stages), (uint32_t)(i / stages) & 1u); ++it)
          __nanosleep(50);
    __syncthreads();
  }

  // Two warps to a lane quarter: they take chunks of tokens in turn (one warp a scheduler leaves it waiting for its own
  // results; 33 clocks a token).
  T* out = static_cast<T*>(g.c) + (int64_t)m0 * g.N + n;
  const uint32_t taddr = tmem + ((uint32_t)((warp & 3) * 32) << 16);
  constexpr int kChunk = NT < 32 ? 8 : 16;
  if (splits == 1) {
#pragma unroll 1
    for (int t0 = group * kChunk; t0 < tokens; t0 += 2 * kChunk) {
      uint32_t v[kChunk];
      tmem_ld<kChunk>(taddr + t0, v);
      finish_tokens<T, kChunk>(v, s_scale + t0, s_zero + t0, zeros, ch, out + (int64_t)t0 * g.N, g.N, tokens - t0,
                               !ok);
    }
  } else {
    uint32_t* part = reinterpret_cast<uint32_t*>(gen);     // [token][channel]
#pragma unroll 1
    for (int t0 = group * kChunk; t0 < tokens; t0 += 2 * kChunk) {
      uint32_t v[kChunk];
      tmem_ld<kChunk>(taddr + t0, v);
#pragma unroll
      for (int i = 0; i < kChunk; ++i) part[(t0 + i) * kRows + c] = v[i];
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");         // the bulk copies read what was just written
    __syncthreads();
    cluster_wait();                                        // every CTA of the cluster runs
    if (!Smem::kLandApart) {
      cluster_arrive();                                    // and has no products to form any more
      cluster_wait();
    }
    // lane r sends to CTA r; a CTA whose sums are not whole sends nothing, and the owners' waits expire
    if (warp == 0 && lane < splits && lane != rank && ok) {
      const int from = lane * run, many = min(run, tokens - from);
      if (many > 0)
        copy_to_cta(in_cta(base + Smem::landing(stages, most) + (uint32_t)((rank < lane ? rank : rank - 1) * many * kRows * 4), lane),
                    base + (uint32_t)(from * kRows * 4), (uint32_t)(many * kRows * 4), in_cta(land_bar, lane));
    }
    __syncwarp();
    if (mine > 0 && !bar_wait(land_bar, 0, abort_flag)) {
      // what the others sent lands all the same before this CTA's memory is released
      ok = false;
      for (uint32_t it = 0; it < kSpinLimit && !mbar_test(land_bar, 0); ++it) __nanosleep(50);
    }
    __syncwarp();
    cluster_arrive();                                      // what was sent here is here
    const uint32_t* own = part + first * kRows + c;
    const uint32_t* landed = reinterpret_cast<const uint32_t*>(gen + Smem::landing(stages, most)) + c;
    const int step = mine * kRows;
#pragma unroll 1
    for (int t0 = group * 4; t0 < mine; t0 += 8) {
      // Four tokens at a time, formed before the first store (see finish_tokens).  Behind the run's last token the sums
      // are of whatever lies there, inside shared memory, and are not stored.
      uint32_t sum[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[i] = own[(t0 + i) * kRows];
      const uint32_t* p = landed + t0 * kRows;
#pragma unroll 3
      for (int r = 1; r < splits; ++r, p += step) {
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] += p[i * kRows];
      }
      float y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = min(first + t0 + i, NT - 1);
        y[i] = finish((int)sum[i], s_scale[t], s_zero[t], ch.b_s, ch.b_sum, ch.bias);
        if (!ok) y[i] = __int_as_float(0x7fffffff);
      }
      if (ch.ok) {
        T* to = out + (int64_t)(first + t0) * g.N;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (t0 + i < mine) to[i * (int64_t)g.N] = Elem<T>::from_f(y[i]);
      }
    }
    __syncwarp();
    cluster_wait();                                        // nobody leaves while its sums are on their way
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)kCols) : "memory");
  report_lost(g.status, abort_flag);
}

// ---- large products: two SMs on one 256 x 256 tile ---------------------------------------------------------------
// cta_group::2: a pair of CTAs holds 256 channels x 256 tokens, each SM 128 channels (TMEM lanes) of all 256 tokens; a
// 128-deep k block is 16 KB of weights and 16 KB of tokens per SM, i.e. 128 products per byte that crosses from L2,
// against 64 for the one-SM tile above.  Persistent, one pair per two SMs; six stages; two accumulators of 256 columns, so
// that eight warps finish one tile while the tensor cores work on the next.  Warp 0 of each CTA copies its own operands and
// signals the leader's barrier, warp 1 of the leader issues the MMAs for both, the others finish 128 tokens of 32
// channels each (sixteen warps with 64 each were 3 % slower: they take issue slots and power from the product).
// Bound by the power limit: 16384 x 4096 x 11008 takes 523 us in a long run (2.8 PFLOP/s, twice what cuBLAS sustains in
// bf16; 389 us with operands of zeros), 2048 x 11008 x 4096 62 us (3.0 PFLOP/s, the tensor pipe 85 % busy).
// The kernel asks for all of an SM's shared memory: no other CTA that needs tensor memory can then lie beside it and
// wait for its columns while it waits for theirs.
constexpr int kPairRows = 256, kPairTokens = 256, kPairStages = 6, kPairBufs = 2;
constexpr int kHalfBytes = 128 * kBlockK;                   // 128 rows of either operand
constexpr int kPairStageBytes = 2 * kHalfBytes;
constexpr int kFinishWarps = 8, kPairThreads = 64 + 32 * kFinishWarps;
constexpr int kPairScales = kPairStages * kPairStageBytes + 256;      // behind the stages and barriers: 1 KB a warp
static_assert(1024 + kPairScales + kFinishWarps * 1024 <= kSmemMost, "");

__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void umma_i8_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}"
      ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(acc)
      : "memory");
}
// arrives on the same barrier of both CTAs
__device__ __forceinline__ void umma_commit_pair(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
      ::"r"(bar), "h"((uint16_t)3)
      : "memory");
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}

struct PairTiles {
  int n_tiles, m_tiles, tokens_first;      // tokens_first: consecutive tiles differ in their tokens
};

template <typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
pair_kernel(const __grid_constant__ Maps maps, Int8Args g, PairTiles pt) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t bar0 = base + kPairStages * kPairStageBytes;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(gen + kPairStages * kPairStageBytes + 8 * (2 * kPairStages + 2 * kPairBufs + 1));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (kPairStages + s); };
  auto acc_full = [&](int b) { return bar0 + 8u * (2 * kPairStages + b); };
  auto acc_empty = [&](int b) { return bar0 + 8u * (2 * kPairStages + kPairBufs + b); };
  const uint32_t retired = bar0 + 8u * (2 * kPairStages + 2 * kPairBufs);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = blockIdx.x & 1u;
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int blocks = (g.K + kBlockK - 1) / kBlockK;
  const int tiles = pt.n_tiles * pt.m_tiles;
  auto origin = [&](int t, int& n0, int& m0) {
    const int a = t % (pt.tokens_first ? pt.m_tiles : pt.n_tiles), b = t / (pt.tokens_first ? pt.m_tiles : pt.n_tiles);
    n0 = (pt.tokens_first ? b : a) * kPairRows;
    m0 = (pt.tokens_first ? a : b) * kPairTokens;
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < kPairStages; ++s) {
      mbar_init(full_bar(s), 1);                  // the leader's: its producer's arrival and both CTAs' bytes
      mbar_init(empty_bar(s), 1);
    }
    for (int b = 0; b < kPairBufs; ++b) {
      mbar_init(acc_full(b), 1);
      mbar_init(acc_empty(b), 2 * kFinishWarps);  // the leader's: the finishing warps of both CTAs
    }
    mbar_init(retired, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"((uint32_t)(kPairBufs * kPairTokens))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tcgen05_fence_before();
  __syncthreads();
  cluster_arrive();                               // the peer's barriers exist before anything is sent to them
  cluster_wait();
  tcgen05_fence_after();
  const uint32_t tmem = *tmem_slot;
  let_next_begin();
  grid_dependency_wait();

  uint32_t issued = 0;                            // k blocks requested (thread 0)
  if (warp == 0) {
    if (lane == 0) {
      int s = 0;
      uint32_t ph = 1;
      bool ok = true;
      const uint32_t full0 = in_cta(full_bar(0), 0);
      for (int t = pair; ok && t < tiles; t += pairs) {
        int n0, m0;
        origin(t, n0, m0);
        n0 += (int)rank * 128, m0 += (int)rank * 128;
        for (int kb = 0; kb < blocks; ++kb) {
          if (!bar_wait(empty_bar(s), ph, abort_flag)) { ok = false; break; }
          const uint32_t sa = base + s * kPairStageBytes;
          if (rank == 0) mbar_expect_tx(full_bar(s), 2 * kPairStageBytes);
          tma_load_pair(sa, &maps.w, kb * kBlockK, n0, full0 + 8u * s);
          tma_load_pair(sa + kHalfBytes, &maps.x, kb * kBlockK, m0, full0 + 8u * s);
          ++issued;
          if (++s == kPairStages) s = 0, ph ^= 1u;
        }
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {
      // the whole warp walks, one lane issues (see stream_kernel)
      int s = 0, buf = 0;
      uint32_t ph = 0, aph = 1;
      bool ok = true;
      const uint64_t dw0 = make_desc_mn_sw128(base, 16, 1024), dx0 = make_desc_mn_sw128(base + kHalfBytes, 16, 1024);
      for (int t = pair; ok && t < tiles; t += pairs) {
        if (!warp_wait(acc_empty(buf), aph, abort_flag)) break;
        tcgen05_fence_after();
        const uint32_t acc = tmem + (uint32_t)(buf * kPairTokens);
        for (int kb = 0; kb < blocks; ++kb) {
          if (!warp_wait(full_bar(s), ph, abort_flag)) { ok = false; break; }
          tcgen05_fence_after();
          const uint64_t at = (uint64_t)(s * (kPairStageBytes >> 4));
          if (elect_one()) {
#pragma unroll
            for (int j = 0; j < kBlockK / 32; ++j)
              umma_i8_pair(acc, dw0 + at + j * 2, dx0 + at + j * 2, idesc_i8(kPairRows, kPairTokens), (kb | j) ? 1u : 0u);
            umma_commit_pair(empty_bar(s));
          }
          __syncwarp();
          if (++s == kPairStages) s = 0, ph ^= 1u;
        }
        if (elect_one()) umma_commit_pair(acc_full(buf));
        __syncwarp();
        if (++buf == kPairBufs) buf = 0, aph ^= 1u;
      }
      if (__any_sync(0xffffffffu, *abort_flag)) {
        // the MMAs already issued retire before the tensor memory is freed
        if (elect_one()) umma_commit_pair(retired);
        for (uint32_t it = 0; it < kSpinLimit && !mbar_test(retired, 0); ++it) __nanosleep(50);
      }
    }
  } else {
    const int q = warp & 3, h = (warp - 2) >> 2;            // TMEM lane quarter; half of the tile's tokens
    // each warp keeps the scales and zero points of its 128 tokens to itself
    float* s_scale = reinterpret_cast<float*>(gen + kPairScales) + (warp - 2) * 256;
    int* s_zero = reinterpret_cast<int*>(s_scale + 128);
    int buf = 0;
    uint32_t aph = 0;
    bool ok = true;
    for (int t = pair; t < tiles; t += pairs) {
      int n0, m0;
      origin(t, n0, m0);
      const int n = n0 + (int)rank * 128 + q * 32 + lane;
      const Channel ch = load_channel<T>(g, n);
      const int mt = m0 + h * 128, tokens = min(128, g.M - mt);
#pragma unroll
      for (int i = lane; i < 128; i += 32) {
        s_scale[i] = i < tokens ? g.a_s[mt + i] : 0.f;
        if (g.a_z) s_zero[i] = i < tokens ? g.a_z[mt + i] : 0;
      }
      __syncwarp();
      // once a wait has expired, the tiles that remain are written as NaN
      ok = ok && warp_wait(acc_full(buf), aph, abort_flag) && __all_sync(0xffffffffu, *abort_flag == 0);
      tcgen05_fence_after();
      const uint32_t taddr = tmem + (uint32_t)(buf * kPairTokens + h * 128) + ((uint32_t)(q * 32) << 16);
      T* out = static_cast<T*>(g.c) + (int64_t)mt * g.N + n;
#pragma unroll 1
      for (int t0 = 0; t0 < tokens; t0 += 32) {
        uint32_t v[32];
        tmem_ld32_nowait(taddr + t0, v);
        tmem_wait_ld();
        finish_tokens<T, 32>(v, s_scale + t0, s_zero + t0, g.a_z != nullptr, ch, out + (int64_t)t0 * g.N, g.N, tokens - t0, !ok);
      }
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(in_cta(acc_empty(buf), 0));
      if (++buf == kPairBufs) buf = 0, aph ^= 1u;
    }
  }

  __syncwarp();
  __syncthreads();
  const bool lost = *abort_flag != 0;
  if (lost && threadIdx.x == 0 && rank == 0) {
    // the copies still in flight (both CTAs') land before shared memory is released
    for (uint32_t i = issued > kPairStages ? issued - kPairStages : 0; i < issued; ++i)
      for (uint32_t it = 0; it < kSpinLimit && !mbar_test(full_bar(i % kPairStages), (i / kPairStages) & 1u); ++it)
        __nanosleep(50);
  }
  report_lost(g.status, abort_flag);
  tcgen05_fence_before();
  __syncthreads();
  cluster_arrive();
  cluster_wait();                                 // no CTA leaves while the other may still signal it or read its operands
  tcgen05_fence_after();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)(kPairBufs * kPairTokens))
                 : "memory");
}

// Self-test of warp_wait.  Nothing arrives on bars[1]; half of the lanes wait on bars[0], whose phase is over, half on
// bars[1], and the flag is raised by another warp a millisecond later: no lane may report the stage as there.  Then a wait on
// bars[0] by all lanes, which succeeds although the flag is raised, and one on bars[1], which the flag ends.
__global__ void wait_selftest_kernel(int32_t* status, uint32_t* answers) {
  __shared__ uint64_t bars[2];
  __shared__ int flag;
  volatile int* abort_flag = &flag;
  if (threadIdx.x == 0) {
    mbar_init(smem_u32(bars), 1);
    mbar_init(smem_u32(bars + 1), 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    mbar_arrive(smem_u32(bars));
  }
  __syncthreads();
  const int lane = threadIdx.x & 31;
  if (threadIdx.x < 32) {
    if (lane == 0) {
      for (int i = 0; i < 1000; ++i) __nanosleep(1000);
      *abort_flag = 1;
    }
  } else {
    const bool some = warp_wait(smem_u32(bars + (lane & 1)), 0, abort_flag);
    const uint32_t a = __ballot_sync(0xffffffffu, some);
    const bool there = warp_wait(smem_u32(bars), 0, abort_flag);
    const uint32_t b = __ballot_sync(0xffffffffu, there);
    const bool never = warp_wait(smem_u32(bars + 1), 0, abort_flag);
    const uint32_t c = __ballot_sync(0xffffffffu, never);
    if (lane == 0) answers[0] = a, answers[1] = b, answers[2] = c;
  }
  __syncthreads();
  report_lost(status, abort_flag);
}

// Self-test of report_lost: the last thread's wait is given up, the reporting thread's succeeds.
__global__ void report_selftest_kernel(int32_t* status) {
  __shared__ uint64_t bars[2];
  __shared__ int flag;
  volatile int* abort_flag = &flag;
  if (threadIdx.x == 0) {
    mbar_init(smem_u32(bars), 1);
    mbar_init(smem_u32(bars + 1), 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    mbar_arrive(smem_u32(bars));
  }
  __syncthreads();
  if (threadIdx.x != blockDim.x - 1) bar_wait(smem_u32(bars), 0, abort_flag);
  else bar_wait(smem_u32(bars + 1), 0, abort_flag);
  __syncthreads();
  report_lost(status, abort_flag);
}

int encode_codes(CUtensorMap* m, const int8_t* p, int64_t k, int64_t rows, int64_t ld, int box_rows) {
  EncodeTiledFn encode = get_encode_fn();
  if (!encode) return LC_ERR_CUDA;
  const cuuint64_t dim[2] = {(cuuint64_t)k, (cuuint64_t)rows};
  const cuuint64_t stride[1] = {(cuuint64_t)ld};
  const cuuint32_t box[2] = {kBlockK, (cuuint32_t)box_rows};
  const cuuint32_t step[2] = {1, 1};
  if (encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t*>(p), dim, stride, box, step,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return LC_ERR_CUDA;
  return LC_OK;
}

// ---- which tile, which split ---------------------------------------------------------------------------------------
// The product of every choice is the same to the bit, so the choice is the one whose estimated time is least.  Fitted to
// measured times (us) of every choice at 378 sizes, M 1 - 6000 and N, K 64 - 11008: a CTA of the first kernel takes `base`
// for its launch, its first copies and its finishing, and c1 for a k block when it has an SM to itself, c2 when two share
// one, in proportion when more come; each CTA that an SM runs besides costs `share` of finishing, and `round` where its
// shared memory lets it begin only after others; splitting K adds the exchange of partial sums.  A wave of pairs takes
// 0.26 a block, or what its finishing takes.  No choice is faster than the weights arrive from HBM, for which many CTAs ask
// sooner than few.  The one taken was 0.8 % behind the best in the mean, within 12 % at all but three sizes of under 9 us
// (e.g. 24 x 4096 x 11008: 11.4 us split eight ways on 32-token tiles, 13.2 four ways on 16-token ones; 256 x 4096 x 4096:
// 10.3 on 64-token tiles, 11.2 on 32-token ones; 1024 x 4096 x 11008: 32 on pairs, 40 on 128-token tiles).
struct Choice {
  int tokens;      // of a tile: 16, 32, 64, 128; 256 for the pair kernel
  int splits;
};
// CTAs that run at once, one to an SM; clusters leave SMs of a GPC over (15 of eight CTAs fit, 33 of four)
constexpr int ctas_at_once(int splits) {
  return splits <= 2 ? kNumSMsB200 : splits <= 6 ? kNumSMsB200 - 16 : kNumSMsB200 - 36;
}
// of clusters, two to an SM
constexpr int kClusteredCtas = 264;

Choice choose(int64_t M, int64_t N, int64_t K) {
  constexpr int kNT[4] = {16, 32, 64, 128};
  constexpr float kBase[4] = {3.1f, 3.4f, 3.4f, 4.5f}, kC1[4] = {0.25f, 0.215f, 0.23f, 0.235f},
                  kC2[4] = {0.26f, 0.315f, 0.39f, 0.41f}, kExchange[4] = {2.0f, 1.6f, 2.9f, 4.0f},
                  kShare[4] = {0.48f, 0.385f, 0.8f, 1.06f}, kRound[4] = {0.45f, 0.6f, 1.3f, 1.0f};
  constexpr int kSplits[6] = {1, 2, 3, 4, 6, 8};
  const int64_t blocks = (K + kBlockK - 1) / kBlockK, n_tiles = (N + kRows - 1) / kRows;
  const float arrive = 4.1f + (float)(N * K) / 6.7e6f;
  Choice best{256, 1};
  const int64_t pair_tiles = ((N + 255) / 256) * ((M + 255) / 256), halves = kNumSMsB200 / 2;
  const float wave = (float)blocks * 0.26f;
  float least = 5.5f + (float)((pair_tiles + halves - 1) / halves) * (wave > 2.8f ? wave : 2.8f);
  if (M <= 128) least = 1e30f;
  for (int i = 0; i < 4; ++i) {
    if (i > 0 && kNT[i - 1] >= M) break;                   // half of the tile's tokens would not exist
    const int64_t m_tiles = (M + kNT[i] - 1) / kNT[i], tiles = n_tiles * m_tiles;
    if (m_tiles > 65535) continue;                         // a grid's second dimension
    for (int sp : kSplits) {
      const int64_t ctas = tiles * sp, count = (blocks + sp - 1) / sp;
      if (sp > 1 && (sp > blocks || ctas > (kNT[i] == 128 ? ctas_at_once(sp) : kClusteredCtas))) break;
      // CTAs that an SM's shared memory holds at once: two when they have more stages than that leaves
      const int64_t fit = kSmemMost / (count * (kWeightBytes + kNT[i] * kBlockK) + 2500);
      const int64_t hold = fit < 2 ? 2 : fit > 4 ? 4 : fit, per_sm = (ctas + kNumSMsB200 - 1) / kNumSMsB200;
      const int64_t rounds = (ctas + hold * kNumSMsB200 - 1) / (hold * kNumSMsB200);
      float t = kBase[i] + (float)(rounds - 1) * kRound[i] + (sp > 1 ? kExchange[i] : 0.f);
      if (ctas <= ctas_at_once(sp)) t += (float)count * kC1[i];
      else t += (float)count * kC2[i] * (per_sm > 2 ? 0.5f * (float)per_sm : 1.f) + (float)(per_sm - 1) * kShare[i];
      if (N * K > (4 << 20)) {
        const float wait = 1.f - (float)ctas / (2.f * kNumSMsB200);
        const float floor = arrive + (sp > 1 ? 0.24f * kExchange[i] : 0.f) + (wait > 0.f ? 0.26f * wait : 0.f);
        if (t < floor) t = floor;
      }
      if (t < least) {
        least = t;
        best = Choice{kNT[i], sp};
      }
    }
  }
  return best;
}

// Whether lc_int8_linear's product quantises the activations itself: one token that a CTA's registers hold.  Its codes are
// 2 KB a k block, 64 KB at most, and leave room for the weights.  (One token of any length gets the 16-token tile.)
bool quantises_itself(int64_t M, int64_t K) { return M == 1 && K <= kMostToken; }

// What a kernel may ask for; the same for every launch, so that calls from two threads do not take it from one another.
template <typename F>
cudaError_t allow_smem(F* kernel) {
  return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMost);
}

template <typename T, int NT, bool kQuant = false>
int launch_stream(const Int8Args& g, int splits, cudaStream_t st) {
  const int n_tiles = (g.N + kRows - 1) / kRows, m_tiles = (g.M + NT - 1) / NT;
  const int blocks = (g.K + kBlockK - 1) / kBlockK;
  const int per_sm = (int64_t)n_tiles * m_tiles * splits > ctas_at_once(splits) ? 2 : 1;
  using Smem = StreamSmem<NT, kQuant>;
  const int most = (blocks + splits - 1) / splits;         // a CTA's blocks: more stages than that are of no use
  int stages = most;
  while (stages > 1 && Smem::bytes(stages, most, splits > 1) > kSmemMost / per_sm - 1024) --stages;
  if (splits > 1 && stages < Smem::kLeast) stages = Smem::kLeast;
  const int smem = Smem::bytes(stages, most, splits > 1);
  Maps maps;
  int rc;
  if ((rc = encode_codes(&maps.w, g.b, g.K, g.N, g.ldb, kRows)) != LC_OK) return rc;
  if (!kQuant && (rc = encode_codes(&maps.x, g.a, g.K, g.M, g.lda, NT)) != LC_OK) return rc;
  LC_CHECK_CUDA(allow_smem(stream_kernel<T, NT, kQuant>));
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = splits, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(n_tiles * splits), (unsigned)m_tiles);
  cfg.blockDim = dim3(kStreamThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  LC_CHECK_CUDA(cudaLaunchKernelEx(&cfg, stream_kernel<T, NT, kQuant>, maps, g, splits, stages));
  return LC_OK;
}

template <typename T>
int launch_pair(const Int8Args& g, cudaStream_t st) {
  Maps maps;
  int rc;
  if ((rc = encode_codes(&maps.w, g.b, g.K, g.N, g.ldb, 128)) != LC_OK) return rc;
  if ((rc = encode_codes(&maps.x, g.a, g.K, g.M, g.lda, 128)) != LC_OK) return rc;
  PairTiles pt;
  pt.n_tiles = (g.N + kPairRows - 1) / kPairRows;
  pt.m_tiles = (g.M + kPairTokens - 1) / kPairTokens;
  pt.tokens_first = pt.m_tiles <= pt.n_tiles;
  const int64_t tiles = (int64_t)pt.n_tiles * pt.m_tiles;
  if (tiles > 0x3fffffff) return LC_ERR_SHAPE;
  const int pairs = (int)(tiles < kNumSMsB200 / 2 ? tiles : kNumSMsB200 / 2);
  LC_CHECK_CUDA(allow_smem(pair_kernel<T>));
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * pairs));
  cfg.blockDim = dim3(kPairThreads);
  cfg.dynamicSmemBytes = kSmemMost;
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  LC_CHECK_CUDA(cudaLaunchKernelEx(&cfg, pair_kernel<T>, maps, g, pt));
  return LC_OK;
}

template <typename T>
int launch(const Int8Args& g, cudaStream_t st) {
  const Choice c = choose(g.M, g.N, g.K);
  switch (c.tokens) {
    case 16: return launch_stream<T, 16>(g, c.splits, st);
    case 32: return launch_stream<T, 32>(g, c.splits, st);
    case 64: return launch_stream<T, 64>(g, c.splits, st);
    case 128: return launch_stream<T, 128>(g, c.splits, st);
    default: return launch_pair<T>(g, st);
  }
}

// sizes, pitches and alignment of the product; the same rules for both entry points
int check(int64_t M, int64_t N, int64_t K, const void* b, int64_t ldb, const float* b_s, bool zeros,
          const int32_t* b_sum, const void* c, int64_t out_dtype) {
  if (out_dtype < LC_F32 || out_dtype > LC_F16 || M < 0 || N < 0 || K <= 0) return LC_ERR_ARG;
  if (zeros && N > 0 && !b_sum) return LC_ERR_ARG;
  // |sum| <= 128 * 128 * K without and 255 * 128 * K with zero points must fit 32 bits
  if (K > (zeros ? 65793 : 131071) || M > (1 << 30) || N > (1 << 30)) return LC_ERR_SHAPE;
  if (M == 0 || N == 0) return LC_OK;
  if (!b || !b_s || !c || ldb < K) return LC_ERR_ARG;
  if (!aligned16(b) || !aligned16(c) || (ldb & 15)) return LC_ERR_ALIGN;
  return LC_OK;
}

// kind::i8 exists on sm_100 only
int check_arch() {
  int dev = 0, major = 0, minor = 0;
  LC_CHECK_CUDA(cudaGetDevice(&dev));
  LC_CHECK_CUDA(cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev));
  LC_CHECK_CUDA(cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, dev));
  return major == 10 && minor == 0 ? LC_OK : LC_ERR_ARCH;
}

int product(const Int8Args& g, int out_dtype, cudaStream_t st) {
  const int rc = check_arch();
  if (rc != LC_OK) return rc;
  switch (out_dtype) {
    case LC_F32: return launch<float>(g, st);
    case LC_BF16: return launch<__nv_bfloat16>(g, st);
    default: return launch<__half>(g, st);
  }
}

}  // namespace
}  // namespace lc

extern "C" LC_API int lc_int8_gemm(const lc_int8_gemm_args* args_host, lc_stream_t stream) {
  using namespace lc;
  if (!args_host) return LC_ERR_ARG;
  const lc_int8_gemm_args& p = *args_host;
  const int rc = check(p.M, p.N, p.K, p.b, p.ldb, p.b_s, p.a_z != nullptr, p.b_sum, p.c, p.out_dtype);
  if (rc != LC_OK || p.M == 0 || p.N == 0) return rc;
  if (!p.a || !p.a_s || p.lda < p.K) return LC_ERR_ARG;
  if (!aligned16(p.a) || (p.lda & 15)) return LC_ERR_ALIGN;
  return product(Int8Args{nullptr, 0, 0, p.a, p.b, p.a_s, p.a_z, p.b_s, p.b_sum, p.bias, p.c, p.status, p.lda, p.ldb, (int)p.M,
                          (int)p.N, (int)p.K},
                 (int)p.out_dtype, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" LC_API int64_t lc_int8_linear_scratch(int64_t M, int64_t K) {
  if (M <= 0 || K <= 0 || lc::quantises_itself(M, K)) return 0;
  return M * ((K + 15) / 16 * 16 + 8);
}

extern "C" LC_API int lc_int8_linear(const lc_int8_linear_args* args_host, lc_stream_t stream) {
  using namespace lc;
  if (!args_host) return LC_ERR_ARG;
  const lc_int8_linear_args& p = *args_host;
  int rc = check(p.M, p.N, p.K, p.b, p.ldb, p.b_s, !p.sym, p.b_sum, p.c, p.dtype);
  if (rc != LC_OK || p.M == 0 || p.N == 0) return rc;
  if (!p.x || p.ldx < 0) return LC_ERR_ARG;
  const int64_t room = lc_int8_linear_scratch(p.M, p.K);
  if (room > 0 && !p.scratch) return LC_ERR_ARG;
  if (p.scratch_bytes < room) return LC_ERR_WORKSPACE;
  if (!aligned16(p.scratch)) return LC_ERR_ALIGN;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int dtype = (int)p.dtype;
  Int8Args g{p.x, p.sym != 0, aligned16(p.x), nullptr, p.b, nullptr, nullptr, p.b_s, p.sym ? nullptr : p.b_sum, p.bias, p.c,
             p.status, 0, p.ldb, (int)p.M, (int)p.N, (int)p.K};
  if (room == 0) {
    if ((rc = check_arch()) != LC_OK) return rc;
    const int splits = choose(1, p.N, p.K).splits;
    switch (dtype) {
      case LC_F32: return launch_stream<float, 16, true>(g, splits, st);
      case LC_BF16: return launch_stream<__nv_bfloat16, 16, true>(g, splits, st);
      default: return launch_stream<__half, 16, true>(g, splits, st);
    }
  }
  const int64_t lda = (p.K + 15) / 16 * 16;
  int8_t* codes = static_cast<int8_t*>(p.scratch);
  float* a_s = reinterpret_cast<float*>(codes + p.M * lda);
  int32_t* a_z = p.sym ? nullptr : reinterpret_cast<int32_t*>(a_s + p.M);
  if ((rc = int8_quant_rows(p.x, dtype, p.M, p.K, p.ldx, codes, lda, a_s, a_z, st)) != LC_OK) return rc;
  g.a = codes, g.lda = lda, g.a_s = a_s, g.a_z = a_z;
  return product(g, dtype, st);
}

extern "C" LC_API int lc_selftest_int8_wait(int32_t* status, uint32_t* answers, lc_stream_t stream) {
  using namespace lc;
  if (!status || !answers) return LC_ERR_ARG;
  wait_selftest_kernel<<<1, 64, 0, reinterpret_cast<cudaStream_t>(stream)>>>(status, answers);
  report_selftest_kernel<<<1, 96, 0, reinterpret_cast<cudaStream_t>(stream)>>>(status + 1);
  LC_LAUNCH_CHECK();
  return LC_OK;
}
