// Products in 8-bit integers: 16- or 32-bit activations [outer, K, inner] quantised
// with one scale per token (outer, inner position), times 8-bit weights [N, K] with one
// scale per output channel, plus bias, to [outer, N, inner].
//
//   m_t = max(max_k |x[t, k]|, 127 * 2^-126), s_t = m_t / 127,
//   q[t, k] = rint(x[t, k] * (127 / m_t)),
//   y[t, j] = float(sum_k q[t, k] w[j, k]) * s_t * s_j + b_j.
//
// The lower bound on m_t keeps 127 / m_t finite: a token of zeros gives q = 0 and y = b.
// The integer sum is exact (K <= 131072 keeps it inside 32 bits); the rest is fp32,
// rounded once to y's type.  A token that holds an infinity or a NaN has no scale:
// its q are 0 and its s_t is infinite or NaN, so that its whole output row is NaN.
#include "plan.h"

namespace mednext {
namespace {

constexpr float kTinyMax = 127.f * 1.17549435e-38f;
constexpr int kI8MaxK = 131072;

// The largest magnitude of a token as ordered bits: the bits of |x| as an unsigned
// number order as |x| does, infinity above every number and NaN above infinity.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

struct TokenScale {
  float scale;    // s_t
  float inverse;  // 127 / m_t, 0 where m_t is not finite
};
__device__ __forceinline__ TokenScale token_scale(uint32_t max_bits) {
  TokenScale s;
  const float m = max_bits >= 0x7f800000u ? __uint_as_float(max_bits) : fmaxf(__uint_as_float(max_bits), kTinyMax);
  s.scale = __fdiv_rn(m, 127.f);
  s.inverse = max_bits >= 0x7f800000u ? 0.f : __fdiv_rn(127.f, m);
  return s;
}
__device__ __forceinline__ int8_t quantize(float v, TokenScale s) {
  // |v| <= m_t, so the product is at most 127 (1 + 2^-23) and rounds into range; a token
  // without a scale gives 0 (inverse 0; infinity * 0 = NaN converts to 0)
  return (int8_t)__float2int_rn(__fmul_rn(v, s.inverse));
}

// One token per warp at a time; inner apart are its elements.
template <typename T>
__global__ void __launch_bounds__(256) i8_quantize_kernel(const T* __restrict__ x, int8_t* __restrict__ q,
                                                          float* __restrict__ scale, long long tokens,
                                                          long long inner, int K, long long pitch) {
  const int lane = threadIdx.x & 31;
  for (long long t = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); t < tokens; t += (long long)gridDim.x * 8) {
    const long long o = t / inner;
    const T* p = x + o * K * inner + (t - o * inner);
    uint32_t m = 0;
    for (int k = lane; k < K; k += 32) m = max(m, abs_bits(to_acc<T>(p[k * inner])));
    m = __reduce_max_sync(0xffffffffu, m);
    const TokenScale s = token_scale(m);
    for (int k = lane; k < pitch; k += 32)
      q[t * pitch + k] = k < K ? quantize(to_acc<T>(p[k * inner]), s) : (int8_t)0;
    if (lane == 0) scale[t] = s.scale;
  }
}

// 64 tokens x 64 outputs per CTA, 64 of K at a time through shared memory.
template <typename T>
__global__ void __launch_bounds__(256) i8_product_kernel(const int8_t* __restrict__ q, const float* __restrict__ qs,
                                                         long long q_pitch, const int8_t* __restrict__ w,
                                                         const float* __restrict__ ws, long long w_pitch,
                                                         const float* __restrict__ bias, T* __restrict__ y,
                                                         long long tokens, long long inner, int K, int N) {
  __shared__ int as[64][17], bs[64][17];
  const long long t0 = (long long)blockIdx.x * 64;
  const int j0 = blockIdx.y * 64;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  int acc[4][4] = {};
  for (int k0 = 0; k0 < K; k0 += 64) {
    for (int i = threadIdx.x; i < 64 * 64; i += 256) {
      const int r = i >> 6, k = i & 63;
      const bool in = k0 + k < K;
      reinterpret_cast<int8_t*>(as[r])[k] = in && t0 + r < tokens ? q[(t0 + r) * q_pitch + k0 + k] : (int8_t)0;
      reinterpret_cast<int8_t*>(bs[r])[k] = in && j0 + r < N ? w[(long long)(j0 + r) * w_pitch + k0 + k] : (int8_t)0;
    }
    __syncthreads();
    for (int k = 0; k < 16; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(as[tx + 16 * i][k], bs[ty + 16 * j][k], acc[i][j]);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const long long t = t0 + tx + 16 * i;
    if (t >= tokens) continue;
    const long long o = t / inner, v = t - o * inner;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = j0 + ty + 16 * j;
      if (n < N)
        y[(o * N + n) * inner + v] =
            from_acc<T>(fmaf((float)acc[i][j] * qs[t], ws[n], bias != nullptr ? bias[n] : 0.f));
    }
  }
}

long long pitch16(int64_t k) { return (k + 15) / 16 * 16; }

template <typename T>
int launch_quantize(const void* x, int8_t* q, float* scale, long long outer, int K, long long inner, long long pitch,
                    cudaStream_t s) {
  const long long tokens = outer * inner;
  i8_quantize_kernel<T><<<(unsigned)std::min<long long>((tokens + 7) / 8, 148 * 16), 256, 0, s>>>(
      static_cast<const T*>(x), q, scale, tokens, inner, K, pitch);
  return record_launch();
}

template <typename T>
int launch_linear(const void* x, const int8_t* w, const float* ws, long long w_pitch, const float* bias, void* y,
                  int8_t* q, float* qs, long long outer, int K, long long inner, int N, cudaStream_t s) {
  int st = launch_quantize<T>(x, q, qs, outer, K, inner, pitch16(K), s);
  if (st != MEDNEXT_OK) return st;
  const long long tokens = outer * inner;
  i8_product_kernel<T><<<dim3((unsigned)((tokens + 63) / 64), (N + 63) / 64), 256, 0, s>>>(
      q, qs, pitch16(K), w, ws, w_pitch, bias, static_cast<T*>(y), tokens, inner, K, N);
  return record_launch();
}

int i8_check(int64_t outer, int64_t k, int64_t inner, int dtype) {
  if (dtype != MEDNEXT_FLOAT32 && dtype != MEDNEXT_BFLOAT16 && dtype != MEDNEXT_FLOAT16) return MEDNEXT_ERR_BAD_DTYPE;
  if (outer < 0 || inner < 0 || k <= 0 || k > kI8MaxK) return MEDNEXT_ERR_BAD_SHAPE;
  const int64_t lim = (int64_t)1 << 30;  // tokens: TMA coordinates and grid sizes are 32-bit
  if (outer > lim || inner > lim || outer * inner > lim) return MEDNEXT_ERR_BAD_SHAPE;
  return MEDNEXT_OK;
}
bool off(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a != 0; }

}  // namespace
}  // namespace mednext

using namespace mednext;

int mednext_int8_quantize(const void* x, int8_t* q, float* scale, int64_t outer, int64_t k, int64_t inner,
                          int64_t q_pitch, int dtype, mednext_stream_t stream) {
  const int st = i8_check(outer, k, inner, dtype);
  if (st != MEDNEXT_OK) return st;
  if (q_pitch < k || q_pitch % 16 != 0 || q_pitch > ((int64_t)1 << 30)) return MEDNEXT_ERR_BAD_SHAPE;
  if (outer * inner == 0) return MEDNEXT_OK;
  if (x == nullptr || q == nullptr || scale == nullptr) return MEDNEXT_ERR_NULL_POINTER;
  if (off(x, elem_size(dtype)) || off(q, 16) || off(scale, 4)) return MEDNEXT_ERR_ALIGNMENT;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  switch (dtype) {
    case MEDNEXT_FLOAT32: return launch_quantize<float>(x, q, scale, outer, (int)k, inner, q_pitch, s);
    case MEDNEXT_BFLOAT16: return launch_quantize<__nv_bfloat16>(x, q, scale, outer, (int)k, inner, q_pitch, s);
    default: return launch_quantize<__half>(x, q, scale, outer, (int)k, inner, q_pitch, s);
  }
}

// The workspace holds the tokens' 8-bit rows, then their scales.
size_t mednext_int8_linear_workspace_size(int64_t outer, int64_t k, int64_t inner, int64_t n, int dtype) {
  if (i8_check(outer, k, inner, dtype) != MEDNEXT_OK || n <= 0) return 0;
  const size_t tokens = (size_t)(outer * inner);
  return tokens * (size_t)pitch16(k) + (tokens * sizeof(float) + 15) / 16 * 16;
}

int mednext_int8_linear(const void* x, const int8_t* weight, const float* weight_scale, const float* bias, void* y,
                        void* workspace, size_t workspace_bytes, int64_t outer, int64_t k, int64_t inner, int64_t n,
                        int64_t weight_pitch, int dtype, mednext_stream_t stream) {
  const int st = i8_check(outer, k, inner, dtype);
  if (st != MEDNEXT_OK) return st;
  if (n <= 0 || n > ((int64_t)1 << 22) || weight_pitch < k || weight_pitch % 16 != 0 ||
      weight_pitch > ((int64_t)1 << 30))
    return MEDNEXT_ERR_BAD_SHAPE;
  if (outer * inner == 0) return MEDNEXT_OK;
  if (x == nullptr || weight == nullptr || weight_scale == nullptr || y == nullptr) return MEDNEXT_ERR_NULL_POINTER;
  if (off(x, elem_size(dtype)) || off(y, elem_size(dtype)) || off(weight, 16) || off(weight_scale, 4) || off(bias, 4))
    return MEDNEXT_ERR_ALIGNMENT;
  if (workspace == nullptr || off(workspace, 16) ||
      workspace_bytes < mednext_int8_linear_workspace_size(outer, k, inner, n, dtype))
    return MEDNEXT_ERR_WORKSPACE;
  int8_t* q = static_cast<int8_t*>(workspace);
  float* qs = reinterpret_cast<float*>(q + (size_t)(outer * inner) * (size_t)pitch16(k));
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  switch (dtype) {
    case MEDNEXT_FLOAT32:
      return launch_linear<float>(x, weight, weight_scale, weight_pitch, bias, y, q, qs, outer, (int)k, inner, (int)n, s);
    case MEDNEXT_BFLOAT16:
      return launch_linear<__nv_bfloat16>(x, weight, weight_scale, weight_pitch, bias, y, q, qs, outer, (int)k, inner,
                                          (int)n, s);
    default:
      return launch_linear<__half>(x, weight, weight_scale, weight_pitch, bias, y, q, qs, outer, (int)k, inner, (int)n, s);
  }
}
