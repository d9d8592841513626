// 8-bit integer linear: C[m][n] = (sum_k (A[m][k] - a_z[m]) B[n][k]) * a_s[m] * b_s[n] (+ bias[n]), A (M x K) int8
// codes of the activations with a scale (and zero point) per token, B (N x K) int8 weights with a scale per
// output channel: the product behind the reference's VllmQuantLinearInt8
// (llmc/compression/quantization/module_utils.py:145-209).
//
// The sum of products is a whole number held exactly in 32 bits, so its value depends neither on the tile nor on
// how the contraction is split; the zero point enters as -a_z[m] * b_sum[n] in the same 32-bit arithmetic (the
// bounds on K keep the final sum inside 32 bits; what wraps on the way wraps back).  After that there are two
// fp32 multiplications and an addition, in this order, and one rounding to the output type.
#include "lc_common.cuh"

namespace lc {

int int8_quant_rows(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ldx, int8_t* codes, int64_t ldc,
                    float* scales, int32_t* zeros, cudaStream_t st);

namespace {

struct Int8Args {
  const int8_t* a;
  const int8_t* b;
  const float* a_s;
  const int32_t* a_z;      // NULL: no zero points
  const float* b_s;
  const int32_t* b_sum;
  const void* bias;        // out_dtype, or NULL
  void* c;                 // [M][N]
  int64_t lda, ldb;
  int M, N, K;
};

// one element of the output; acc is the sum of the products of the codes
template <typename T>
__device__ __forceinline__ float finish(int acc, float a_s, int a_z, float b_s, int b_sum, float bias) {
  const int whole = (int)((unsigned)acc - (unsigned)a_z * (unsigned)b_sum);
  return __fadd_rn(__fmul_rn(__fmul_rn(__int2float_rn(whole), a_s), b_s), bias);
}

constexpr int kTile = 64, kThreads = 256;

// 64 x 64 outputs per CTA, 4 x 4 per thread, four products per DP4A
template <typename T>
__global__ void __launch_bounds__(kThreads) dp4a_kernel(Int8Args g) {
  __shared__ uint32_t sa[kTile][17], sb[kTile][17];
  const int m0 = blockIdx.y * kTile, n0 = blockIdx.x * kTile;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int lr = threadIdx.x >> 2, lc = (threadIdx.x & 3) * 16;       // row and first byte this thread stages
  int acc[4][4] = {};
  auto stage = [&](const int8_t* p, int64_t ld, int row, int rows, int k0, uint32_t* dst) {
    uint32_t w[4] = {0u, 0u, 0u, 0u};
    const int k = k0 + lc;
    if (row < rows && k < g.K) {
      const int8_t* src = p + (int64_t)row * ld + k;
      if (k + 16 <= g.K) {
        const uint4 v = *reinterpret_cast<const uint4*>(src);
        w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
      } else {
        for (int i = 0; i < g.K - k; ++i) w[i >> 2] |= (uint32_t)(uint8_t)src[i] << (8 * (i & 3));
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) dst[i] = w[i];
  };
  for (int k0 = 0; k0 < g.K; k0 += 64) {
    stage(g.a, g.lda, m0 + lr, g.M, k0, &sa[lr][lc >> 2]);
    stage(g.b, g.ldb, n0 + lr, g.N, k0, &sb[lr][lc >> 2]);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      int av[4], bv[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) av[i] = (int)sa[ty + 16 * i][k], bv[i] = (int)sb[tx + 16 * i][k];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(av[i], bv[j], acc[i][j]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int n = n0 + tx + 16 * j;
    if (n >= g.N) continue;
    const float bs = g.b_s[n], bias = g.bias ? Elem<T>::to_f(static_cast<const T*>(g.bias)[n]) : 0.f;
    const int bsum = g.a_z ? g.b_sum[n] : 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int m = m0 + ty + 16 * i;
      if (m < g.M)
        static_cast<T*>(g.c)[(int64_t)m * g.N + n] =
            Elem<T>::from_f(finish<T>(acc[i][j], g.a_s[m], g.a_z ? g.a_z[m] : 0, bs, bsum, bias));
    }
  }
}

template <typename T>
int launch(const Int8Args& g, cudaStream_t st) {
  const dim3 grid((unsigned)((g.N + kTile - 1) / kTile), (unsigned)((g.M + kTile - 1) / kTile));
  if (grid.y > 65535) return LC_ERR_SHAPE;
  dp4a_kernel<T><<<grid, kThreads, 0, st>>>(g);
  LC_LAUNCH_CHECK();
  return LC_OK;
}

// sizes, pitches and alignment of the product; the same rules for both entry points
int check(int64_t M, int64_t N, int64_t K, const void* b, int64_t ldb, const float* b_s, bool zeros,
          const int32_t* b_sum, const void* c, int out_dtype) {
  if (out_dtype < LC_F32 || out_dtype > LC_F16 || M < 0 || N < 0 || K <= 0) return LC_ERR_ARG;
  if (zeros && N > 0 && !b_sum) return LC_ERR_ARG;
  // |sum| <= 128 * 128 * K without and 255 * 128 * K with zero points must fit 32 bits
  if (K > (zeros ? 65793 : 131071) || M > (1 << 30) || N > (1 << 30)) return LC_ERR_SHAPE;
  if (M == 0 || N == 0) return LC_OK;
  if (!b || !b_s || !c || ldb < K) return LC_ERR_ARG;
  if (!aligned16(b) || !aligned16(c) || (ldb & 15)) return LC_ERR_ALIGN;
  return LC_OK;
}

int product(const Int8Args& g, int out_dtype, cudaStream_t st) {
  switch (out_dtype) {
    case LC_F32: return launch<float>(g, st);
    case LC_BF16: return launch<__nv_bfloat16>(g, st);
    default: return launch<__half>(g, st);
  }
}

}  // namespace
}  // namespace lc

extern "C" LC_API int lc_int8_gemm(const int8_t* a, int64_t lda, const float* a_s, const int32_t* a_z, const int8_t* b,
                                   int64_t ldb, const float* b_s, const int32_t* b_sum, const void* bias, int64_t M,
                                   int64_t N, int64_t K, void* c, int out_dtype, int32_t* status, lc_stream_t stream) {
  using namespace lc;
  (void)status;
  const int rc = check(M, N, K, b, ldb, b_s, a_z != nullptr, b_sum, c, out_dtype);
  if (rc != LC_OK || M == 0 || N == 0) return rc;
  if (!a || !a_s || lda < K) return LC_ERR_ARG;
  if (!aligned16(a) || (lda & 15)) return LC_ERR_ALIGN;
  return product(Int8Args{a, b, a_s, a_z, b_s, b_sum, bias, c, lda, ldb, (int)M, (int)N, (int)K}, out_dtype,
                 reinterpret_cast<cudaStream_t>(stream));
}

extern "C" LC_API int64_t lc_int8_linear_scratch(int64_t M, int64_t K) {
  if (M < 0 || K < 0) return 0;
  return M * ((K + 15) / 16 * 16) + 8 * M;
}

extern "C" LC_API int lc_int8_linear(const void* x, int dtype, int64_t ldx, const int8_t* b, int64_t ldb, const float* b_s,
                                     const int32_t* b_sum, const void* bias, int64_t M, int64_t N, int64_t K, int sym,
                                     void* c, void* scratch, int64_t scratch_bytes, int32_t* status, lc_stream_t stream) {
  using namespace lc;
  (void)status;
  const int rc = check(M, N, K, b, ldb, b_s, !sym, b_sum, c, dtype);
  if (rc != LC_OK || M == 0 || N == 0) return rc;
  if (!x || ldx < 0 || !scratch) return LC_ERR_ARG;
  if (scratch_bytes < lc_int8_linear_scratch(M, K)) return LC_ERR_WORKSPACE;
  if (!aligned16(scratch)) return LC_ERR_ALIGN;
  const int64_t lda = (K + 15) / 16 * 16;
  int8_t* codes = static_cast<int8_t*>(scratch);
  float* a_s = reinterpret_cast<float*>(codes + M * lda);
  int32_t* a_z = sym ? nullptr : reinterpret_cast<int32_t*>(a_s + M);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int qrc = int8_quant_rows(x, dtype, M, K, ldx, codes, lda, a_s, a_z, st);
  if (qrc != LC_OK) return qrc;
  return product(Int8Args{codes, b, a_s, a_z, b_s, b_sum, bias, c, lda, ldb, (int)M, (int)N, (int)K}, dtype, st);
}
