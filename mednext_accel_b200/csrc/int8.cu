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
#include <cstring>

#include "plan.h"
#include "pointwise_tma.cuh"
#include "tma_host.h"

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

// ------------------------------ quantisation ------------------------------
// Four values of one token to four bytes.
__device__ __forceinline__ uint32_t quantize4(float a, float b, float c, float d, TokenScale s) {
  return (uint32_t)(uint8_t)quantize(a, s) | (uint32_t)(uint8_t)quantize(b, s) << 8 |
         (uint32_t)(uint8_t)quantize(c, s) << 16 | (uint32_t)(uint8_t)quantize(d, s) << 24;
}

// Any layout and width: one token per warp at a time, inner apart its elements, which are
// read twice.
template <typename T>
__global__ void __launch_bounds__(256) i8_quantize_any_kernel(const T* __restrict__ x, int8_t* __restrict__ q,
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

// ------------------------------ the product on the tensor cores ------------------------------
// D[128 rows of A, bn rows of B] = A B^T in 8-bit integers with 32-bit sums
// (tcgen05.mma kind::i8), both operands K-major rows under a 128-byte swizzle.
//
// Which operand is A goes by the output's layout, so that the 32 lanes of an accumulator
// column lie side by side in y: channels-first output takes the tokens as A (lane =
// voxel), rows take the weights as A (lane = output channel).
//
// Persistent, warp-specialised: warp 0 issues the TMA loads (a ring of 128-byte K
// blocks), warp 1 owns TMEM and issues the MMAs into two accumulators in turn, warps 2-9
// scale and store.  The waits and the exit follow the pointwise kernels' discipline: every wait
// is bounded, and what is in flight is waited for before TMEM is freed.
constexpr int kI8BM = 128, kI8BK = 128;
constexpr int kI8Threads = 320, kI8EpiWarps = 8;
constexpr int kI8MaxStages = 8;

struct I8GemmArgs {
  const float* a_scale;  // of A's rows
  const float* b_scale;  // of B's rows
  const float* bias;     // of the output channels, or NULL
  void* y;
  int a_rows, b_rows, K;
  int inner;  // of y
  int N;      // output channels
  int bn, stages, a_tiles, b_tiles;
};

struct I8Shared {
  uint64_t full[kI8MaxStages], empty[kI8MaxStages];
  uint64_t tfull[2], tempty[2];
  uint64_t drain;
  uint32_t tmem_base;
  int abort;
  float2 col[kI8EpiWarps][32];  // (scale, bias) of an epilogue warp's 32 columns
};

// Instruction descriptor, kind::i8: signed 8-bit operands, K-major, 32-bit integer sums.
__host__ __device__ constexpr uint32_t make_idesc_i8(int M, int N) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ void mma_i8_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                          uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

template <typename T, bool TOKENS_A>
__global__ void __launch_bounds__(kI8Threads, 1)
    i8_gemm_kernel(const __grid_constant__ CUtensorMap mA, const __grid_constant__ CUtensorMap mB, I8GemmArgs p) {
  extern __shared__ uint8_t i8_raw[];
  __shared__ I8Shared sh;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* ringA = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(i8_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* ringB = ringA + (size_t)p.stages * (kI8BM * kI8BK);
  const int b_bytes = p.bn * kI8BK;
  const uint32_t tmem_cols = (uint32_t)(2 * p.bn);
  if (warp == 1) tmem_alloc(&sh.tmem_base, tmem_cols);
  if (threadIdx.x == 0) {
    for (int i = 0; i < p.stages; ++i) {
      mbar_init(&sh.full[i], 1);
      mbar_init(&sh.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.tfull[i], 1);
      mbar_init(&sh.tempty[i], kI8EpiWarps * 32);
    }
    mbar_init(&sh.drain, 1);
    sh.abort = 0;
    fence_mbarrier_init();
    tma_prefetch_map(&mA);
    tma_prefetch_map(&mB);
  }
  if (warp == 1) tmem_relinquish();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem_base;
  volatile int* abort = &sh.abort;
  const int tiles = p.a_tiles * p.b_tiles;
  const int mine = (tiles - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x;
  const int kblocks = (p.K + kI8BK - 1) / kI8BK;
  long long issued = 0;
  // neighbouring CTAs share a tile of tokens and differ in the output channels
  const auto decode = [&](int i, int& a0, int& b0) {
    const int t = (int)blockIdx.x + i * (int)gridDim.x;
    const int ta = TOKENS_A ? t / p.b_tiles : t % p.a_tiles, tb = TOKENS_A ? t % p.b_tiles : t / p.a_tiles;
    a0 = ta * kI8BM;
    b0 = tb * p.bn;
  };

  if (warp == 0) {
    if (lane == 0) {
      bool ok = true;
      for (int i = 0; i < mine && ok; ++i) {
        int a0, b0;
        decode(i, a0, b0);
        for (int kb = 0; kb < kblocks; ++kb) {
          const int st = (int)(issued % p.stages);
          const long long turn = issued / p.stages;
          if (turn > 0 && !(ok = wait_or_abort(&sh.empty[st], (uint32_t)((turn - 1) & 1), abort))) break;
          mbar_arrive_expect_tx(&sh.full[st], (uint32_t)(kI8BM * kI8BK + b_bytes));
          tma_load_2d(ringA + (size_t)st * (kI8BM * kI8BK), &mA, &sh.full[st], kb * kI8BK, a0);
          tma_load_2d(ringB + (size_t)st * b_bytes, &mB, &sh.full[st], kb * kI8BK, b0);
          ++issued;
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = make_idesc_i8(kI8BM, p.bn);
      long long q = 0;
      bool ok = true;
      for (int i = 0; i < mine && ok; ++i) {
        const int acc = i & 1;
        if (i >= 2 && !wait_or_abort(&sh.tempty[acc], (uint32_t)(((i >> 1) - 1) & 1), abort)) break;
        tc_fence_after();
        const uint32_t d = tmem + (uint32_t)(acc * p.bn);
        for (int kb = 0; kb < kblocks; ++kb, ++q) {
          const int st = (int)(q % p.stages);
          if (!(ok = wait_or_abort(&sh.full[st], (uint32_t)((q / p.stages) & 1), abort))) break;
          tc_fence_after();
          const uint32_t sa = smem_u32(ringA + (size_t)st * (kI8BM * kI8BK)), sb = smem_u32(ringB + (size_t)st * b_bytes);
          const int steps = min(kI8BK, p.K - kb * kI8BK + 31) / 32;  // 32 of K per instruction; zeros past K
          for (int ks = 0; ks < steps; ++ks)
            mma_i8_ss(d, make_sw128_desc(sa + ks * 32, 16, 1024), make_sw128_desc(sb + ks * 32, 16, 1024), idesc,
                      kb > 0 || ks > 0 ? 1u : 0u);
          mma_commit(&sh.empty[st]);
        }
        if (ok) mma_commit(&sh.tfull[acc]);
      }
    }
  } else {
    // accumulator lanes 32 * (warp % 4) ..; the two groups of four warps take turns at the
    // 32-column pieces
    const int q4 = warp & 3, half = (warp - 2) >> 2;
    float2* col = sh.col[warp - 2];
    for (int i = 0; i < mine; ++i) {
      const int acc = i & 1;
      if (!__all_sync(0xffffffffu, wait_or_abort(&sh.tfull[acc], (uint32_t)((i >> 1) & 1), abort))) break;
      tc_fence_after();
      int a0, b0;
      decode(i, a0, b0);
      const int row = a0 + q4 * 32 + lane;
      const bool in = row < p.a_rows;
      float row_scale = 0.f, row_bias = 0.f;
      T* y = static_cast<T*>(p.y);
      long long step;  // from one column to the next
      if (in) row_scale = p.a_scale[row];
      if (TOKENS_A) {
        const int o = row / p.inner;
        y += ((long long)o * p.N + b0) * p.inner + (row - o * p.inner);
        step = p.inner;
      } else {
        if (in && p.bias != nullptr) row_bias = p.bias[row];
        y += (long long)b0 * p.N + row;
        step = p.N;
      }
      for (int c0 = half * 32; c0 < p.bn && b0 + c0 < p.b_rows; c0 += 64) {
        const int c = b0 + c0 + lane;
        uint32_t r[32];
        __syncwarp();  // whole again, and the previous piece's constants are read
        tmem_ld32(tmem + (uint32_t)(acc * p.bn + c0) + ((uint32_t)(q4 * 32) << 16), r);
        col[lane] = c < p.b_rows ? make_float2(p.b_scale[c], TOKENS_A && p.bias != nullptr ? p.bias[c] : 0.f)
                                 : make_float2(0.f, 0.f);
        __syncwarp();
        tmem_ld_wait();
        T* at = y + c0 * step;
        const int n = min(32, p.b_rows - b0 - c0);
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          const float2 k = col[j];
          const float v = (float)(int)r[j];
          // (sum * token's scale) * channel's scale + bias
          if (in && j < n)
            *at = from_acc<T>(TOKENS_A ? fmaf(v * row_scale, k.x, k.y) : fmaf(v * k.x, row_scale, row_bias));
          at += step;
        }
      }
      __syncwarp();
      tc_fence_before();
      mbar_arrive(&sh.tempty[acc]);
    }
  }
  __syncthreads();
  if (*abort && lane == 0) {
    if (warp == 0) drain_ring(sh.full, p.stages, issued);
    if (warp == 1) drain_mma(&sh.drain);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, tmem_cols);
}

int num_sms() {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0)
    return 148;
  return sms;
}

// q: [tokens][q_pitch], w: [N][w_pitch]; y [outer, N, inner]
template <typename T>
int launch_gemm(const int8_t* q, const float* qs, long long q_pitch, const int8_t* w, const float* ws,
                long long w_pitch, const float* bias, void* y, long long tokens, long long inner, int K, int N,
                cudaStream_t s) {
  const bool tokens_a = inner > 1;
  I8GemmArgs p{};
  p.a_scale = tokens_a ? qs : ws;
  p.b_scale = tokens_a ? ws : qs;
  p.bias = bias;
  p.y = y;
  p.a_rows = tokens_a ? (int)tokens : N;
  p.b_rows = tokens_a ? N : (int)tokens;
  p.K = K;
  p.inner = (int)inner;
  p.N = N;
  p.a_tiles = (p.a_rows + kI8BM - 1) / kI8BM;
  const int sms = num_sms();
  // the widest B tile that still gives every SM a tile, at most what B fills
  p.bn = 256;
  while (p.bn > 32 && (p.bn / 2 >= p.b_rows || (long long)p.a_tiles * ((p.b_rows + p.bn - 1) / p.bn) < sms)) p.bn /= 2;
  p.b_tiles = (p.b_rows + p.bn - 1) / p.bn;
  if ((long long)p.a_tiles * p.b_tiles >= ((long long)1 << 31)) return MEDNEXT_ERR_BAD_SHAPE;
  const int stage = kI8BM * kI8BK + p.bn * kI8BK;
  p.stages = std::min(kI8MaxStages, (200 * 1024) / stage);
  const size_t smem = (size_t)p.stages * stage + 1024;
  CUtensorMap mA, mB;
  if (!tma::encode_rows_8bit(&mA, tokens_a ? q : w, K, p.a_rows, tokens_a ? q_pitch : w_pitch, kI8BM) ||
      !tma::encode_rows_8bit(&mB, tokens_a ? w : q, K, p.b_rows, tokens_a ? w_pitch : q_pitch, p.bn)) {
    note_cuda_error(cudaErrorInvalidValue);
    return MEDNEXT_ERR_CUDA;
  }
  const unsigned grid = (unsigned)std::min<long long>((long long)p.a_tiles * p.b_tiles, sms);
  auto run = [&](auto kern) {
    const int st = ensure_smem(kern, smem);
    if (st != MEDNEXT_OK) return st;
    kern<<<grid, kI8Threads, smem, s>>>(mA, mB, p);
    return record_launch();
  };
  return tokens_a ? run(i8_gemm_kernel<T, true>) : run(i8_gemm_kernel<T, false>);
}

long long pitch16(int64_t k) { return (k + 15) / 16 * 16; }

template <typename T>
int launch_quantize(const void* x, int8_t* q, float* scale, long long outer, int K, long long inner, long long pitch,
                    cudaStream_t s) {
  const long long tokens = outer * inner;
  i8_quantize_any_kernel<T><<<(unsigned)std::min<long long>((tokens + 7) / 8, 148 * 16), 256, 0, s>>>(
      static_cast<const T*>(x), q, scale, tokens, inner, K, pitch);
  return record_launch();
}

template <typename T>
int launch_linear(const void* x, const int8_t* w, const float* ws, long long w_pitch, const float* bias, void* y,
                  int8_t* q, float* qs, long long outer, int K, long long inner, int N, cudaStream_t s) {
  int st = launch_quantize<T>(x, q, qs, outer, K, inner, pitch16(K), s);
  if (st != MEDNEXT_OK) return st;
  return launch_gemm<T>(q, qs, pitch16(K), w, ws, w_pitch, bias, y, outer * inner, inner, K, N, s);
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

MEDNEXT_DEFINE_ERROR_READER(read_clear_errors_int8)

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
