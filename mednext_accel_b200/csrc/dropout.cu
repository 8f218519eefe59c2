// Dropout from a counter-based generator, optionally added to a residual:
//   y[i] = residual[i] + (word(i) >= drop ? x[i] * 65536 / (65536 - drop) : 0)
// word(i) is the 16-bit word i % 8 (low half of the first 32-bit output first) of
// Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as
// 1, 2, 3", SC 2011) at counter (i / 8, offset) under the 64-bit key `seed`.  The mask is
// a function of (seed, offset, i) alone: it is never stored, and the backward pass is
// the same map applied to dy.  16 bits per element make one generator call serve one
// 16-byte vector of 16-bit data; the rate is drop / 65536 exactly, and the scale is
// made from that rate, so the mean is kept.
#include "plan.h"

namespace mednext {
namespace {

constexpr int kDropThreads = 256;

struct DropArgs {
  const void* x;
  const void* residual;  // NULL: none
  void* y;
  const int64_t* rng;     // device {seed, offset} added to the two below, or NULL
  uint64_t seed, offset;
  int64_t* used;  // receives {seed, offset} as this launch used them; NULL: not wanted
  long long n;
  uint32_t drop;  // 0..65536
  float scale;
};

__device__ __forceinline__ uint4 philox4x32_10(uint64_t ctr_lo, uint64_t ctr_hi, uint64_t key) {
  uint32_t a = (uint32_t)ctr_lo, b = (uint32_t)(ctr_lo >> 32), c = (uint32_t)ctr_hi, d = (uint32_t)(ctr_hi >> 32);
  uint32_t k0 = (uint32_t)key, k1 = (uint32_t)(key >> 32);
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t p = (uint64_t)0xD2511F53u * a, q = (uint64_t)0xCD9E8D57u * c;
    a = (uint32_t)(q >> 32) ^ b ^ k0;
    b = (uint32_t)q;
    c = (uint32_t)(p >> 32) ^ d ^ k1;
    d = (uint32_t)p;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(a, b, c, d);
}

// A dropped element gives 0 whatever x holds there (infinities and NaN included).
__device__ __forceinline__ float drop_one(uint32_t word, uint32_t drop, float x, float scale) {
  return word >= drop ? __fmul_rn(x, scale) : 0.f;
}

template <typename T>
__global__ void __launch_bounds__(kDropThreads) dropout_kernel(DropArgs a) {
  uint64_t seed = a.seed, offset = a.offset;
  if (a.rng != nullptr) {
    seed += (uint64_t)a.rng[0];
    offset += (uint64_t)a.rng[1];
  }
  if (a.used != nullptr && blockIdx.x == 0 && threadIdx.x == 0) {
    a.used[0] = (int64_t)seed;
    a.used[1] = (int64_t)offset;
  }
  const T* x = static_cast<const T*>(a.x);
  const T* res = static_cast<const T*>(a.residual);
  T* y = static_cast<T*>(a.y);
  const long long groups = (a.n + 7) / 8;
  for (long long g = (long long)blockIdx.x * kDropThreads + threadIdx.x; g < groups;
       g += (long long)gridDim.x * kDropThreads) {
    const uint4 r = philox4x32_10((uint64_t)g, offset, seed);
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const long long i = g * 8 + j;
      if (i >= a.n) break;
      const uint32_t word = (j & 1) ? w[j >> 1] >> 16 : w[j >> 1] & 0xffffu;
      const float v = drop_one(word, a.drop, to_acc<T>(x[i]), a.scale);
      y[i] = from_acc<T>(res != nullptr ? to_acc<T>(res[i]) + v : v);
    }
  }
}

template <typename T>
int launch_dropout(const DropArgs& a, cudaStream_t s) {
  const long long blocks = ((a.n + 7) / 8 + kDropThreads - 1) / kDropThreads;
  dropout_kernel<T><<<(unsigned)std::min<long long>(blocks, 148 * 16), kDropThreads, 0, s>>>(a);
  return record_launch();
}

}  // namespace
}  // namespace mednext

using namespace mednext;

int mednext_dropout(const void* x, const void* residual, void* y, const int64_t* rng, uint64_t seed, uint64_t offset,
                    int64_t* used, int64_t n, int drop, int dtype, mednext_stream_t stream) {
  if (dtype != MEDNEXT_FLOAT32 && dtype != MEDNEXT_BFLOAT16 && dtype != MEDNEXT_FLOAT16) return MEDNEXT_ERR_BAD_DTYPE;
  if (n < 0 || n > ((int64_t)1 << 48)) return MEDNEXT_ERR_BAD_SHAPE;
  if (drop < 0 || drop > 65536) return MEDNEXT_ERR_BAD_VALUE;
  if (n > 0 && (x == nullptr || y == nullptr)) return MEDNEXT_ERR_NULL_POINTER;
  const size_t esz = elem_size(dtype);
  if ((reinterpret_cast<uintptr_t>(x) % esz) || (reinterpret_cast<uintptr_t>(y) % esz) ||
      (reinterpret_cast<uintptr_t>(residual) % esz) || (reinterpret_cast<uintptr_t>(rng) & 7) ||
      (reinterpret_cast<uintptr_t>(used) & 7))
    return MEDNEXT_ERR_ALIGNMENT;
  if (n == 0) return MEDNEXT_OK;
  DropArgs a{};
  a.x = x; a.residual = residual; a.y = y;
  a.rng = rng; a.seed = seed; a.offset = offset; a.used = used;
  a.n = n; a.drop = (uint32_t)drop;
  a.scale = drop == 65536 ? 0.f : 65536.f / (float)(65536 - drop);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  switch (dtype) {
    case MEDNEXT_FLOAT32: return launch_dropout<float>(a, s);
    case MEDNEXT_BFLOAT16: return launch_dropout<__nv_bfloat16>(a, s);
    default: return launch_dropout<__half>(a, s);
  }
}
