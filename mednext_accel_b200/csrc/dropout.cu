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

// The words of U groups, a block's worth of threads apart: counters (hi, lo + u * threads).
// The rounds run side by side, so that each round key is made once.  `hi`, the offset and the
// keys are the same in every thread of the CTA: the first products of them are too.
template <int U>
__device__ __forceinline__ void philox4x32_10(uint32_t lo, uint32_t hi, uint64_t offset, uint64_t key,
                                              uint32_t (&w)[U][4]) {
  uint32_t k0 = (uint32_t)key, k1 = (uint32_t)(key >> 32);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    w[u][0] = lo + u * kDropThreads;
    w[u][1] = hi;
    w[u][2] = (uint32_t)offset;
    w[u][3] = (uint32_t)(offset >> 32);
  }
#pragma unroll
  for (int i = 0; i < 10; ++i) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint64_t p = (uint64_t)0xD2511F53u * w[u][0], q = (uint64_t)0xCD9E8D57u * w[u][2];
      w[u][0] = (uint32_t)(q >> 32) ^ w[u][1] ^ k0;
      w[u][1] = (uint32_t)q;
      w[u][2] = (uint32_t)(p >> 32) ^ w[u][3] ^ k1;
      w[u][3] = (uint32_t)p;
    }
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
}

// x scale where the word's low (high) 16 bits reach drop, else 0 whatever x holds
// (infinities and NaN included).  threshold = drop << 16; none: drop = 65536.
struct DropRule {
  uint32_t threshold;
  bool none;
  float scale;
  __device__ __forceinline__ float2 pair(uint32_t word, float2 x) const {
    const float2 v = __fmul2_rn(x, make_float2(scale, scale));
    return make_float2((word << 16) >= threshold && !none ? v.x : 0.f, word >= threshold && !none ? v.y : 0.f);
  }
};

// Eight elements, one generator call, per group; U groups per thread, their loads issued
// before the generator runs.  VEC: every tensor starts on 16 bytes, and CTAs whose groups
// are all whole move 16-byte vectors; RES: a residual is added.  One turn per CTA.
//
// 67.1 M bf16 elements: with a residual 61.7 us, 6.5 TB/s, bound by HBM; without 47.7 us, 5.6
// TB/s, bound by instructions too: about 5 per element for the generator (4 a round) and 5
// for the rest against 4 bytes of traffic.  One group per thread took 55.7 us: U = 4 shares
// the round keys and keeps 64 bytes of x in flight.  Tensors off 16 bytes move single elements: 172 us with a residual.
template <typename T, bool VEC, bool RES, int U>
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
  const DropRule rule{a.drop << 16, a.drop == 65536u, a.scale};
  constexpr int kVecs = (int)sizeof(T) / 2;  // vectors per group
  constexpr int kPer = 8 / kVecs;            // elements per vector
  constexpr uint32_t kGroups = kDropThreads * U;  // per CTA; a power of two
  // the CTA's first group: a multiple of kGroups, so that no thread's low word carries
  const uint64_t g0 = (uint64_t)blockIdx.x * kGroups;
  const uint32_t lo = (uint32_t)g0 + threadIdx.x, hi = (uint32_t)(g0 >> 32);
  const long long first = (long long)(g0 + threadIdx.x) * 8;
  const T* x = static_cast<const T*>(a.x) + first;
  const T* res = static_cast<const T*>(a.residual) + first;
  T* y = static_cast<T*>(a.y) + first;
  uint32_t w[U][4];
  if (VEC && (long long)(g0 + kGroups) * 8 <= a.n) {
    uint4 qx[U][kVecs], qr[U][kVecs];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int v = 0; v < kVecs; ++v) {
        qx[u][v] = reinterpret_cast<const uint4*>(x + u * kDropThreads * 8)[v];
        if (RES) qr[u][v] = reinterpret_cast<const uint4*>(res + u * kDropThreads * 8)[v];
      }
    philox4x32_10<U>(lo, hi, offset, seed, w);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int v = 0; v < kVecs; ++v) {
        float f[kPer], add[kPer];
        unpack16<T>(qx[u][v], f);
        if (RES) unpack16<T>(qr[u][v], add);
#pragma unroll
        for (int i = 0; i < kPer; i += 2) {
          float2 t = rule.pair(w[u][(v * kPer + i) / 2], make_float2(f[i], f[i + 1]));
          if (RES) t = __fadd2_rn(make_float2(add[i], add[i + 1]), t);
          f[i] = t.x;
          f[i + 1] = t.y;
        }
        reinterpret_cast<uint4*>(y + u * kDropThreads * 8)[v] = pack16<T>(f);
      }
    return;
  }
  philox4x32_10<U>(lo, hi, offset, seed, w);
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int at = u * kDropThreads * 8 + j;
      if (first + at >= a.n) continue;
      const float f = to_acc<T>(x[at]);
      const float2 t = rule.pair(w[u][j >> 1], make_float2(f, f));
      const float v = (j & 1) ? t.y : t.x;
      y[at] = from_acc<T>(RES ? to_acc<T>(res[at]) + v : v);
    }
}

template <typename T, bool VEC, bool RES, int U>
int launch_dropout_as(const DropArgs& a, cudaStream_t s) {
  const long long ctas = ((a.n + 7) / 8 + kDropThreads * U - 1) / (kDropThreads * U);
  dropout_kernel<T, VEC, RES, U><<<(unsigned)ctas, kDropThreads, 0, s>>>(a);
  return record_launch();
}
template <typename T, bool RES>
int launch_dropout_for(const DropArgs& a, cudaStream_t s) {
  const uintptr_t bits = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.y) |
                         reinterpret_cast<uintptr_t>(a.residual);
  constexpr int U = sizeof(T) == 2 ? 4 : 2;  // 64 bytes of x per thread
  if (bits % 16 != 0) return launch_dropout_as<T, false, RES, 1>(a, s);
  // one group per thread while that is all the GPU holds at once
  if (a.n < 148LL * 2048 * 8 * U) return launch_dropout_as<T, true, RES, 1>(a, s);
  return launch_dropout_as<T, true, RES, U>(a, s);
}
template <typename T>
int launch_dropout(const DropArgs& a, cudaStream_t s) {
  return a.residual != nullptr ? launch_dropout_for<T, true>(a, s) : launch_dropout_for<T, false>(a, s);
}

}  // namespace
}  // namespace mednext

using namespace mednext;

int mednext_dropout(const void* x, const void* residual, void* y, const int64_t* rng, uint64_t seed, uint64_t offset,
                    int64_t* used, int64_t n, int drop, int dtype, mednext_stream_t stream) {
  if (dtype != MEDNEXT_FLOAT32 && dtype != MEDNEXT_BFLOAT16 && dtype != MEDNEXT_FLOAT16) return MEDNEXT_ERR_BAD_DTYPE;
  if (n < 0 || n > ((int64_t)1 << 40)) return MEDNEXT_ERR_BAD_SHAPE;
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
