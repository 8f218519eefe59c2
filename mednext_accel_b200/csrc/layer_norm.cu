// Layer norm over one axis of a contiguous [outer, C, inner] tensor, forward and
// backward.  inner = 1 is the last-axis form ([tokens, C] rows); inner > 1 is the
// channels-first form, one token per (outer, inner) position, its channels inner
// elements apart (NCDHW volumes, one token per voxel).
//
//   mean = sum x / C, var = sum (x - mean)^2 / C, r = (var + eps)^-1/2,
//   xh = (x - mean) r, y = xh w + b;
//   g = dy w, dx = r (g - mean(g) - xh mean(g xh)), dw = sum dy xh, db = sum dy.
//
// Statistics and all sums are fp32 (the final fold of the weight-grad partials fp64);
// each output is rounded once, to its own type.  The variance is summed about the mean,
// so a mean far larger than the spread costs no digits.  Every sum has a fixed order:
// results are the same bits from call to call.
#include "plan.h"

namespace mednext {
namespace {

constexpr int kSms = 148;

struct LnArgs {
  const void* x;
  const void* dy;
  const void* w;  // NULL: ones
  const void* b;  // NULL: zeros
  void* y;        // forward: y; backward: dx
  float2* stats;  // per token (mean, r); forward: NULL when not wanted
  float* part;    // backward: [parts][2][C] weight-grad partials (NULL when not wanted)
  long long outer, inner, tokens;
  int C;
  int pdt;  // parameter dtype
  float eps;
};

__device__ __forceinline__ float load_param(const void* p, int dtype, int i, float none) {
  if (p == nullptr) return none;
  if (dtype == MEDNEXT_FLOAT32) return static_cast<const float*>(p)[i];
  if (dtype == MEDNEXT_BFLOAT16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}

// Sums of two values over the CTA, the same in every thread; red: 2 * 32 floats.
__device__ __forceinline__ float2 cta_sum2(float a, float b, float2* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  __syncthreads();  // the previous call's sums may still be read
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = make_float2(a, b);
  __syncthreads();
  float2 s = red[0];
  for (int w = 1; w < (int)(blockDim.x >> 5); ++w) {
    s.x += red[w].x;
    s.y += red[w].y;
  }
  return s;
}

// ------------------------------ any width, rows ------------------------------
// One CTA per row at a time; the row is read again for each pass (from L1 / L2).
template <typename T>
__global__ void __launch_bounds__(256) ln_rows_any_fwd_kernel(LnArgs a) {
  __shared__ float2 red[32];
  for (long long t = blockIdx.x; t < a.tokens; t += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + t * a.C;
    T* y = static_cast<T*>(a.y) + t * a.C;
    float s = 0.f;
    for (int c = threadIdx.x; c < a.C; c += blockDim.x) s += to_acc<T>(x[c]);
    const float mean = cta_sum2(s, 0.f, red).x / (float)a.C;
    s = 0.f;
    for (int c = threadIdx.x; c < a.C; c += blockDim.x) {
      const float d = to_acc<T>(x[c]) - mean;
      s = fmaf(d, d, s);
    }
    const float r = rsqrtf(cta_sum2(s, 0.f, red).x / (float)a.C + a.eps);
    for (int c = threadIdx.x; c < a.C; c += blockDim.x)
      y[c] = from_acc<T>(fmaf((to_acc<T>(x[c]) - mean) * r, load_param(a.w, a.pdt, c, 1.f), load_param(a.b, a.pdt, c, 0.f)));
    if (a.stats != nullptr && threadIdx.x == 0) a.stats[t] = make_float2(mean, r);
  }
}

template <typename T>
__global__ void __launch_bounds__(256) ln_rows_any_dx_kernel(LnArgs a) {
  __shared__ float2 red[32];
  for (long long t = blockIdx.x; t < a.tokens; t += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + t * a.C;
    const T* dy = static_cast<const T*>(a.dy) + t * a.C;
    T* dx = static_cast<T*>(a.y) + t * a.C;
    const float2 st = a.stats[t];
    float s1 = 0.f, s2 = 0.f;
    for (int c = threadIdx.x; c < a.C; c += blockDim.x) {
      const float g = to_acc<T>(dy[c]) * load_param(a.w, a.pdt, c, 1.f);
      s1 += g;
      s2 = fmaf(g, (to_acc<T>(x[c]) - st.x) * st.y, s2);
    }
    const float2 m = cta_sum2(s1, s2, red);
    const float m1 = m.x / (float)a.C, m2 = m.y / (float)a.C;
    for (int c = threadIdx.x; c < a.C; c += blockDim.x) {
      const float g = to_acc<T>(dy[c]) * load_param(a.w, a.pdt, c, 1.f);
      dx[c] = from_acc<T>(st.y * (g - m1 - (to_acc<T>(x[c]) - st.x) * st.y * m2));
    }
  }
}

// ------------------------------ any width, channels first ------------------------------
// 32 neighbouring tokens per CTA (lanes), 8 warps over the channels.
template <typename T>
__global__ void __launch_bounds__(256) ln_chan_any_fwd_kernel(LnArgs a) {
  __shared__ float red[8][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long per = (a.inner + 31) / 32, tiles = a.outer * per;
  for (long long tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const long long o = tile / per, v = (tile - o * per) * 32 + lane;
    const bool in = v < a.inner;
    const long long base = o * a.C * a.inner + v;
    const T* x = static_cast<const T*>(a.x) + base;
    T* y = static_cast<T*>(a.y) + base;
    float stat[2];
    for (int pass = 0; pass < 2; ++pass) {
      float s = 0.f;
      for (int c = warp; c < a.C; c += 8) {
        const float d = in ? to_acc<T>(x[(long long)c * a.inner]) - (pass ? stat[0] : 0.f) : 0.f;
        s += pass ? d * d : d;
      }
      __syncthreads();
      red[warp][lane] = s;
      __syncthreads();
      s = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) s += red[w][lane];
      stat[pass] = pass ? rsqrtf(s / (float)a.C + a.eps) : s / (float)a.C;
    }
    if (!in) continue;
    for (int c = warp; c < a.C; c += 8)
      y[(long long)c * a.inner] = from_acc<T>(fmaf((to_acc<T>(x[(long long)c * a.inner]) - stat[0]) * stat[1],
                                                   load_param(a.w, a.pdt, c, 1.f), load_param(a.b, a.pdt, c, 0.f)));
    if (a.stats != nullptr && warp == 0) a.stats[o * a.inner + v] = make_float2(stat[0], stat[1]);
  }
}

template <typename T>
__global__ void __launch_bounds__(256) ln_chan_any_dx_kernel(LnArgs a) {
  __shared__ float2 red[8][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long per = (a.inner + 31) / 32, tiles = a.outer * per;
  for (long long tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const long long o = tile / per, v = (tile - o * per) * 32 + lane;
    const bool in = v < a.inner;
    const long long base = o * a.C * a.inner + v;
    const T* x = static_cast<const T*>(a.x) + base;
    const T* dy = static_cast<const T*>(a.dy) + base;
    T* dx = static_cast<T*>(a.y) + base;
    const float2 st = in ? a.stats[o * a.inner + v] : make_float2(0.f, 0.f);
    float2 s = make_float2(0.f, 0.f);
    if (in)
      for (int c = warp; c < a.C; c += 8) {
        const float g = to_acc<T>(dy[(long long)c * a.inner]) * load_param(a.w, a.pdt, c, 1.f);
        s.x += g;
        s.y = fmaf(g, (to_acc<T>(x[(long long)c * a.inner]) - st.x) * st.y, s.y);
      }
    __syncthreads();
    red[warp][lane] = s;
    __syncthreads();
    s = make_float2(0.f, 0.f);
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      s.x += red[w][lane].x;
      s.y += red[w][lane].y;
    }
    const float m1 = s.x / (float)a.C, m2 = s.y / (float)a.C;
    if (in)
      for (int c = warp; c < a.C; c += 8) {
        const float g = to_acc<T>(dy[(long long)c * a.inner]) * load_param(a.w, a.pdt, c, 1.f);
        dx[(long long)c * a.inner] =
            from_acc<T>(st.y * (g - m1 - (to_acc<T>(x[(long long)c * a.inner]) - st.x) * st.y * m2));
      }
  }
}

// ------------------------------ weight-grad partials, any width ------------------------------
// Rows: a CTA owns 32 columns x one part of the tokens, 8 warps striding its rows.
template <typename T>
__global__ void __launch_bounds__(256) ln_rows_any_dw_kernel(LnArgs a, int parts) {
  __shared__ float2 red[8][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane, p = blockIdx.y;
  const long long per = (a.tokens + parts - 1) / parts;
  const long long t0 = p * per, t1 = min(t0 + per, a.tokens);
  float2 s = make_float2(0.f, 0.f);
  if (c < a.C)
    for (long long t = t0 + warp; t < t1; t += 8) {
      const float2 st = a.stats[t];
      const float d = to_acc<T>(static_cast<const T*>(a.dy)[t * a.C + c]);
      s.x = fmaf(d, (to_acc<T>(static_cast<const T*>(a.x)[t * a.C + c]) - st.x) * st.y, s.x);
      s.y += d;
    }
  red[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && c < a.C) {
    for (int w = 1; w < 8; ++w) {
      s.x += red[w][lane].x;
      s.y += red[w][lane].y;
    }
    a.part[((long long)p * 2) * a.C + c] = s.x;
    a.part[((long long)p * 2 + 1) * a.C + c] = s.y;
  }
}

// Channels first: a CTA owns one channel x one part of the tokens.
template <typename T>
__global__ void __launch_bounds__(256) ln_chan_any_dw_kernel(LnArgs a, int parts) {
  __shared__ float2 red[32];
  const int c = blockIdx.x, p = blockIdx.y;
  const long long per = (a.tokens + parts - 1) / parts;
  const long long t0 = p * per, t1 = min(t0 + per, a.tokens);
  float2 s = make_float2(0.f, 0.f);
  for (long long t = t0 + threadIdx.x; t < t1; t += blockDim.x) {
    const long long o = t / a.inner, v = t - o * a.inner, i = (o * a.C + c) * a.inner + v;
    const float2 st = a.stats[t];
    const float d = to_acc<T>(static_cast<const T*>(a.dy)[i]);
    s.x = fmaf(d, (to_acc<T>(static_cast<const T*>(a.x)[i]) - st.x) * st.y, s.x);
    s.y += d;
  }
  s = cta_sum2(s.x, s.y, red);
  if (threadIdx.x == 0) {
    a.part[((long long)p * 2) * a.C + c] = s.x;
    a.part[((long long)p * 2 + 1) * a.C + c] = s.y;
  }
}

__device__ __forceinline__ void store_param(void* p, int dtype, int i, double v) {
  if (p == nullptr) return;
  if (dtype == MEDNEXT_FLOAT32) static_cast<float*>(p)[i] = (float)v;
  else if (dtype == MEDNEXT_BFLOAT16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn((float)v);
  else static_cast<__half*>(p)[i] = __float2half_rn((float)v);
}

// dw, db = the partials' sums in a fixed order: 32 warps take every 32nd part of 32
// columns, then one adds the 32 sums.  parts = 0 writes zeros (no tokens).
__global__ void __launch_bounds__(1024) ln_fold_kernel(const float* __restrict__ part, int parts, int C, void* dw,
                                                      void* db, int pdt) {
  __shared__ double red[2][32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  double s0 = 0.0, s1 = 0.0;
  if (c < C)
#pragma unroll 8
    for (int p = warp; p < parts; p += 32) {
      s0 += (double)part[((long long)p * 2) * C + c];
      s1 += (double)part[((long long)p * 2 + 1) * C + c];
    }
  red[0][warp][lane] = s0;
  red[1][warp][lane] = s1;
  __syncthreads();
  if (warp == 0 && c < C) {
    for (int w = 1; w < 32; ++w) {
      s0 += red[0][w][lane];
      s1 += red[1][w][lane];
    }
    store_param(dw, pdt, c, s0);
    store_param(db, pdt, c, s1);
  }
}

// Makes the compiler take the packed words as new values: it unpacks them again (one
// instruction for two bf16) instead of keeping the unpacked copies in registers.
__device__ __forceinline__ void renew(uint32_t& v) { asm volatile("" : "+r"(v)); }
__device__ __forceinline__ void renew(float& v) {}
__device__ __forceinline__ void renew(__nv_bfloat16& v) { asm volatile("" : "+h"(reinterpret_cast<uint16_t&>(v))); }
__device__ __forceinline__ void renew(__half& v) { asm volatile("" : "+h"(reinterpret_cast<uint16_t&>(v))); }
__device__ __forceinline__ void renew(uint4& q) {
  renew(q.x);
  renew(q.y);
  renew(q.z);
  renew(q.w);
}

// ------------------------------ rows held in registers ------------------------------
// G threads hold a row, EPT elements each, loaded once as 16-byte vectors (VEC elements;
// VEC = 1 where rows do not start on 16 bytes) that stay packed until they are used.
// G <= 32 is a power of two and its sums are shuffles; a larger G is whole warps, which
// add through shared memory, one barrier per sum, R rows' sums at once.
template <typename T, int VEC, int EPT>
struct RowFrag {
  static constexpr int kVecs = EPT / VEC;
  uint4 q[kVecs];
  // column of element 0 of vector v
  static __device__ __forceinline__ int col(int v, int gl, int G) { return (v * G + gl) * VEC; }
  __device__ __forceinline__ void load(const T* row, int gl, int G, int C, bool in) {
#pragma unroll
    for (int v = 0; v < kVecs; ++v) {
      const int c = col(v, gl, G);
      q[v] = in && c < C ? *reinterpret_cast<const uint4*>(row + c) : make_uint4(0, 0, 0, 0);
    }
  }
  __device__ __forceinline__ void get(int v, float* f) const { unpack16<T>(q[v], f); }
  __device__ __forceinline__ void again() {
#pragma unroll
    for (int v = 0; v < kVecs; ++v) renew(q[v]);
  }
  static __device__ __forceinline__ void store(T* row, int c, const float* f) {
    *reinterpret_cast<uint4*>(row + c) = pack16<T>(f);
  }
};
template <typename T, int EPT>
struct RowFrag<T, 1, EPT> {
  static constexpr int kVecs = EPT;
  T e[EPT];
  static __device__ __forceinline__ int col(int v, int gl, int G) { return v * G + gl; }
  __device__ __forceinline__ void load(const T* row, int gl, int G, int C, bool in) {
#pragma unroll
    for (int v = 0; v < EPT; ++v) {
      const int c = v * G + gl;
      e[v] = in && c < C ? row[c] : from_acc<T>(0.f);
    }
  }
  __device__ __forceinline__ void get(int v, float* f) const { f[0] = to_acc<T>(e[v]); }
  __device__ __forceinline__ void again() {
#pragma unroll
    for (int v = 0; v < EPT; ++v) renew(e[v]);
  }
  static __device__ __forceinline__ void store(T* row, int c, const float* f) { row[c] = from_acc<T>(f[0]); }
};

// p + step as a value of its own: the 32 products k * step of an unrolled loop would
// otherwise be kept over the loop about it, 64 registers.
template <typename T>
__device__ __forceinline__ void advance(T*& p, long long step) {
  p += step;
  asm volatile("" : "+l"(p));
}

// Shared-memory loads that stay where they are written: hoisted out of the loop over
// tiles, a thread's parameters would take 32 or 64 registers.
__device__ __forceinline__ float2 lds2(const float2* p) {
  float2 v;
  asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(smem_u32(p)));
  return v;
}
__device__ __forceinline__ float lds1(const float* p) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(smem_u32(p)));
  return v;
}

// Sums of N values over the G threads of a group, the same in each; red holds two
// buffers of N x 32, taken in turn: the barrier of the next sum separates their uses.
template <int N>
__device__ __forceinline__ void group_sum(float (&v)[N], int G, float* red, int& turn) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    if (o < G) {
#pragma unroll
      for (int n = 0; n < N; ++n) v[n] += __shfl_xor_sync(0xffffffffu, v[n], o);
    }
  if (G <= 32) return;
  float* r = red + turn * N * 32;
  turn ^= 1;
  const int warp = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0) {
#pragma unroll
    for (int n = 0; n < N; ++n) r[n * 32 + warp] = v[n];
  }
  __syncthreads();
  const int w0 = (threadIdx.x / G) * (G >> 5), w1 = w0 + (G >> 5);
#pragma unroll
  for (int n = 0; n < N; ++n) v[n] = 0.f;
  for (int w = w0; w < w1; ++w) {
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] += r[n * 32 + w];
  }
}

template <typename T, int VEC, int EPT, int R, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == 256 ? (R > 1 ? 3 : 4) : 1) ln_rows_fwd_kernel(LnArgs a, int G) {
  using Frag = RowFrag<T, VEC, EPT>;
  constexpr int kVecs = Frag::kVecs;
  __shared__ float red[2 * R * 32];
  int turn = 0;
  const int groups = blockDim.x / G, gi = threadIdx.x / G, gl = threadIdx.x - gi * G;
  const float rc = 1.f / (float)a.C;
  // up to 8 columns: the parameters stay in registers over the rows
  float w[EPT <= 8 ? EPT : 1], b[EPT <= 8 ? EPT : 1];
  if (EPT <= 8) {
#pragma unroll
    for (int v = 0; v < kVecs; ++v)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const int c = Frag::col(v, gl, G) + i;
        w[(v * VEC + i) % (EPT <= 8 ? EPT : 1)] = c < a.C ? load_param(a.w, a.pdt, c, 1.f) : 0.f;
        b[(v * VEC + i) % (EPT <= 8 ? EPT : 1)] = c < a.C ? load_param(a.b, a.pdt, c, 0.f) : 0.f;
      }
  }
  for (long long base = (long long)blockIdx.x * groups * R; base < a.tokens; base += (long long)gridDim.x * groups * R) {
    Frag x[R];
    float s[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long t = base + r * groups + gi;
      x[r].load(static_cast<const T*>(a.x) + t * a.C, gl, G, a.C, t < a.tokens);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      s[r] = 0.f;
#pragma unroll
      for (int v = 0; v < kVecs; ++v) {
        float f[VEC];
        x[r].get(v, f);
#pragma unroll
        for (int i = 0; i < VEC; ++i) s[r] += f[i];
      }
    }
    group_sum<R>(s, G, red, turn);
    float mean[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      x[r].again();
      mean[r] = s[r] * rc;
      s[r] = 0.f;
#pragma unroll
      for (int v = 0; v < kVecs; ++v) {
        float f[VEC];
        x[r].get(v, f);
        if (Frag::col(v, gl, G) < a.C) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            const float d = f[i] - mean[r];
            s[r] = fmaf(d, d, s[r]);
          }
        }
      }
    }
    group_sum<R>(s, G, red, turn);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long t = base + r * groups + gi;
      if (t >= a.tokens) continue;
      x[r].again();
      const float rstd = rsqrtf(s[r] * rc + a.eps);
      T* y = static_cast<T*>(a.y) + t * a.C;
#pragma unroll
      for (int v = 0; v < kVecs; ++v) {
        const int c = Frag::col(v, gl, G);
        if (c >= a.C) continue;
        float f[VEC];
        x[r].get(v, f);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float wi = EPT <= 8 ? w[(v * VEC + i) % (EPT <= 8 ? EPT : 1)] : load_param(a.w, a.pdt, c + i, 1.f);
          const float bi = EPT <= 8 ? b[(v * VEC + i) % (EPT <= 8 ? EPT : 1)] : load_param(a.b, a.pdt, c + i, 0.f);
          f[i] = fmaf((f[i] - mean[r]) * rstd, wi, bi);
        }
        Frag::store(y, c, f);
      }
      if (a.stats != nullptr && gl == 0) a.stats[t] = make_float2(mean[r], rstd);
    }
  }
}

// The threads own their columns over all rows of the CTA, so the weight grads are sums
// in registers; the CTA adds its groups' sums through shared memory (acc: [slots][2][C],
// a slot per warp for G <= 32, per group else) and writes one partial per CTA.
template <typename T, int VEC, int EPT, int R, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == 256 ? (R > 1 ? 2 : 3) : 1) ln_rows_bwd_kernel(LnArgs a, int G) {
  using Frag = RowFrag<T, VEC, EPT>;
  constexpr int kVecs = Frag::kVecs;
  extern __shared__ __align__(16) float ln_acc[];
  __shared__ float red[2 * 2 * R * 32];
  int turn = 0;
  const int groups = blockDim.x / G, gi = threadIdx.x / G, gl = threadIdx.x - gi * G;
  const float rc = 1.f / (float)a.C;
  float w[EPT], dw[EPT], db[EPT];
#pragma unroll
  for (int v = 0; v < kVecs; ++v)
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const int c = Frag::col(v, gl, G) + i;
      w[v * VEC + i] = c < a.C ? load_param(a.w, a.pdt, c, 1.f) : 0.f;
      dw[v * VEC + i] = db[v * VEC + i] = 0.f;
    }
  for (long long base = (long long)blockIdx.x * groups * R; base < a.tokens; base += (long long)gridDim.x * groups * R) {
    Frag x[R], d[R];
    float2 st[R];
    float s[2 * R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long t = base + r * groups + gi;
      const bool in = t < a.tokens;
      x[r].load(static_cast<const T*>(a.x) + t * a.C, gl, G, a.C, in);
      d[r].load(static_cast<const T*>(a.dy) + t * a.C, gl, G, a.C, in);
      st[r] = in ? a.stats[t] : make_float2(0.f, 0.f);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      s[2 * r] = s[2 * r + 1] = 0.f;
#pragma unroll
      for (int v = 0; v < kVecs; ++v) {
        float f[VEC], g[VEC];
        x[r].get(v, f);
        d[r].get(v, g);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float xh = (f[i] - st[r].x) * st[r].y, gw = g[i] * w[v * VEC + i];
          dw[v * VEC + i] = fmaf(g[i], xh, dw[v * VEC + i]);
          db[v * VEC + i] += g[i];
          s[2 * r] += gw;
          s[2 * r + 1] = fmaf(gw, xh, s[2 * r + 1]);
        }
      }
    }
    group_sum<2 * R>(s, G, red, turn);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long t = base + r * groups + gi;
      if (t >= a.tokens) continue;
      x[r].again();
      d[r].again();
      const float m1 = s[2 * r] * rc, m2 = s[2 * r + 1] * rc;
      T* dx = static_cast<T*>(a.y) + t * a.C;
#pragma unroll
      for (int v = 0; v < kVecs; ++v) {
        const int c = Frag::col(v, gl, G);
        if (c >= a.C) continue;
        float f[VEC], g[VEC];
        x[r].get(v, f);
        d[r].get(v, g);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float xh = (f[i] - st[r].x) * st[r].y;
          f[i] = st[r].y * (fmaf(g[i], w[v * VEC + i], -m1) - xh * m2);
        }
        Frag::store(dx, c, f);
      }
    }
  }
  if (a.part == nullptr) return;
  // lanes of one warp that hold the same columns, then the CTA's slots, in order
#pragma unroll
  for (int i = 0; i < EPT; ++i)
    for (int o = G; o < 32; o <<= 1) {
      dw[i] += __shfl_xor_sync(0xffffffffu, dw[i], o);
      db[i] += __shfl_xor_sync(0xffffffffu, db[i], o);
    }
  const int slot = G < 32 ? threadIdx.x >> 5 : gi, slots = G < 32 ? blockDim.x >> 5 : groups;
  if (G >= 32 || (threadIdx.x & 31) < G) {
#pragma unroll
    for (int v = 0; v < kVecs; ++v)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const int c = Frag::col(v, gl, G) + i;
        if (c < a.C) {
          ln_acc[(size_t)(2 * slot) * a.C + c] = dw[v * VEC + i];
          ln_acc[(size_t)(2 * slot + 1) * a.C + c] = db[v * VEC + i];
        }
      }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < 2 * a.C; c += blockDim.x) {
    float v = 0.f;
    for (int i = 0; i < slots; ++i) v += ln_acc[(size_t)i * 2 * a.C + c];
    a.part[(long long)blockIdx.x * 2 * a.C + c] = v;
  }
}

// ------------------------------ channels first, held in registers ------------------------------
// A lane owns W neighbouring tokens (one 32-bit word of 16-bit data, W = 2, where rows
// start on words and inner is even; else one element) and CPT channels of them; a tile of
// 32 W tokens takes S = ceil(C / CPT) warps, channel k S + s belonging to warp s.  Each
// load is one coalesced row segment of a channel, and x is read once.  Only two numbers per token cross the
// warps, once per tile.  blockDim = (32, S, P), P tiles per CTA side by side.
template <typename T, int W>
struct Word;
template <typename T>
struct Word<T, 1> {
  T v;
  __device__ __forceinline__ void load(const T* p, bool in) { v = in ? *p : from_acc<T>(0.f); }
  __device__ __forceinline__ void get(float (&f)[1]) const { f[0] = to_acc<T>(v); }
  static __device__ __forceinline__ void store(T* p, const float (&f)[1]) { *p = from_acc<T>(f[0]); }
};
template <typename T>
struct Word<T, 2> {
  uint32_t v;
  __device__ __forceinline__ void load(const T* p, bool in) { v = in ? *reinterpret_cast<const uint32_t*>(p) : 0u; }
  __device__ __forceinline__ void get(float (&f)[2]) const {
    const float2 t = unpack2<T>(v);
    f[0] = t.x;
    f[1] = t.y;
  }
  static __device__ __forceinline__ void store(T* p, const float (&f)[2]) {
    *reinterpret_cast<uint32_t*>(p) = pack2<T>(make_float2(f[0], f[1]));
  }
};

constexpr int kChanCpt = 32;

template <typename T, int W, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == 256 ? 3 : 1) ln_chan_fwd_kernel(LnArgs a) {
  extern __shared__ __align__(16) float2 ln_sm[];  // [C] (w, b), then two buffers [P][S][W][32] (sum, M2)
  const int lane = threadIdx.x, s = threadIdx.y, S = blockDim.y, P = blockDim.z;
  for (int c = threadIdx.x + 32 * (threadIdx.y + S * threadIdx.z); c < a.C; c += 32 * S * P)
    ln_sm[c] = make_float2(load_param(a.w, a.pdt, c, 1.f), load_param(a.b, a.pdt, c, 0.f));
  float2* red = ln_sm + a.C + threadIdx.z * S * W * 32;
  const int buffer = P * S * W * 32;
  int turn = 0;
  __syncthreads();
  const long long per = (a.inner + 32 * W - 1) / (32 * W), tiles = a.outer * per;
  const float rc = 1.f / (float)a.C;
  const int mine = s < a.C ? (a.C - s + S - 1) / S : 0;  // channels of this warp
  for (long long base = (long long)blockIdx.x * P; base < tiles; base += (long long)gridDim.x * P) {
    const long long tile = base + threadIdx.z;
    const long long o = tile / per, v = (tile - o * per) * (32 * W) + lane * W;
    const bool in = tile < tiles && v < a.inner;  // inner is even where W = 2
    const long long at = (o * a.C + s) * a.inner + v, step = (long long)S * a.inner;
    Word<T, W> x[kChanCpt];
    const T* px = static_cast<const T*>(a.x) + at;
#pragma unroll
    for (int k = 0; k < kChanCpt; ++k, advance(px, step)) x[k].load(px, in && k < mine);
    float mean[W], m2[W];
#pragma unroll
    for (int j = 0; j < W; ++j) mean[j] = m2[j] = 0.f;
#pragma unroll
    for (int k = 0; k < kChanCpt; ++k) {
      float f[W];
      x[k].get(f);
#pragma unroll
      for (int j = 0; j < W; ++j) mean[j] += f[j];
    }
    if (S == 1) {
#pragma unroll
      for (int j = 0; j < W; ++j) mean[j] *= rc;
    } else {
      // the warp's own mean for its own squares; both join below (Chan, Golub and LeVeque)
      const float rm = mine > 0 ? 1.f / (float)mine : 0.f;
#pragma unroll
      for (int j = 0; j < W; ++j) mean[j] *= rm;
    }
#pragma unroll
    for (int k = 0; k < kChanCpt; ++k)
      if (k < mine) {
        float f[W];
        renew(x[k].v);
        x[k].get(f);
#pragma unroll
        for (int j = 0; j < W; ++j) m2[j] = fmaf(f[j] - mean[j], f[j] - mean[j], m2[j]);
      }
    if (S > 1) {
      float2* r = red + turn * buffer;
      turn ^= 1;
#pragma unroll
      for (int j = 0; j < W; ++j) r[(s * W + j) * 32 + lane] = make_float2(mean[j], m2[j]);
      __syncthreads();
#pragma unroll
      for (int j = 0; j < W; ++j) {
        float sum = 0.f, sq = 0.f;
        for (int i = 0; i < S; ++i) sum = fmaf((float)((a.C - i + S - 1) / S), r[(i * W + j) * 32 + lane].x, sum);
        mean[j] = sum * rc;
        for (int i = 0; i < S; ++i) {
          const float2 p = r[(i * W + j) * 32 + lane];
          const float d = p.x - mean[j];
          sq += fmaf((float)((a.C - i + S - 1) / S) * d, d, p.y);
        }
        m2[j] = sq;
      }
    }
    float rstd[W];
#pragma unroll
    for (int j = 0; j < W; ++j) rstd[j] = rsqrtf(m2[j] * rc + a.eps);
    if (in) {
      T* y = static_cast<T*>(a.y) + at;
#pragma unroll
      for (int k = 0; k < kChanCpt; ++k, advance(y, step))
        if (k < mine) {
          const float2 wb = lds2(ln_sm + k * S + s);
          float f[W];
          renew(x[k].v);
          x[k].get(f);
#pragma unroll
          for (int j = 0; j < W; ++j) f[j] = fmaf((f[j] - mean[j]) * rstd[j], wb.x, wb.y);
          Word<T, W>::store(y, f);
        }
      if (a.stats != nullptr && s == 0) {
#pragma unroll
        for (int j = 0; j < W; ++j) a.stats[o * a.inner + v + j] = make_float2(mean[j], rstd[j]);
      }
    }
  }
}

// Sums over the 32 lanes of 32 values each: lane l returns the sum of value l.  Halves
// change places at distances 16, 8, ..., 1: 31 shuffles instead of 160.
__device__ __forceinline__ float transpose_sum(float (&v)[32], int lane) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const bool up = lane & o;
#pragma unroll
    for (int i = 0; i < o; ++i) {
      const float send = up ? v[i] : v[i + o], keep = up ? v[i + o] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
    }
  }
  return v[0];
}

template <typename T, int W, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == 256 ? 2 : 1) ln_chan_bwd_kernel(LnArgs a) {
  extern __shared__ __align__(16) float2 ln_sm[];  // [C] (w, -), then two buffers [P][S][W][32] of sums
  const int lane = threadIdx.x, s = threadIdx.y, S = blockDim.y, P = blockDim.z;
  float* wsm = reinterpret_cast<float*>(ln_sm);
  for (int c = threadIdx.x + 32 * (threadIdx.y + S * threadIdx.z); c < a.C; c += 32 * S * P)
    wsm[c] = load_param(a.w, a.pdt, c, 1.f);
  float2* red = ln_sm + a.C + threadIdx.z * S * W * 32;
  const int buffer = P * S * W * 32;
  int turn = 0;
  __syncthreads();
  const long long per = (a.inner + 32 * W - 1) / (32 * W), tiles = a.outer * per;
  const float rc = 1.f / (float)a.C;
  const int mine = s < a.C ? (a.C - s + S - 1) / S : 0;
  float dw = 0.f, db = 0.f;  // of channel lane * S + s
  for (long long base = (long long)blockIdx.x * P; base < tiles; base += (long long)gridDim.x * P) {
    const long long tile = base + threadIdx.z;
    const long long o = tile / per, v = (tile - o * per) * (32 * W) + lane * W;
    const bool in = tile < tiles && v < a.inner;
    const long long at = (o * a.C + s) * a.inner + v, step = (long long)S * a.inner;
    Word<T, W> x[kChanCpt], d[kChanCpt];
    const T *px = static_cast<const T*>(a.x) + at, *pd = static_cast<const T*>(a.dy) + at;
#pragma unroll
    for (int k = 0; k < kChanCpt; ++k, advance(px, step), advance(pd, step)) {
      x[k].load(px, in && k < mine);
      d[k].load(pd, in && k < mine);
    }
    float2 st[W], sum[W];
#pragma unroll
    for (int j = 0; j < W; ++j) {
      st[j] = in ? a.stats[o * a.inner + v + j] : make_float2(0.f, 0.f);
      sum[j] = make_float2(0.f, 0.f);
    }
#pragma unroll
    for (int k = 0; k < kChanCpt; ++k)
      if (k < mine) {
        const float w = lds1(wsm + k * S + s);
        float f[W], g[W];
        x[k].get(f);
        d[k].get(g);
#pragma unroll
        for (int j = 0; j < W; ++j) {
          const float gw = g[j] * w;
          sum[j].x += gw;
          sum[j].y = fmaf(gw, (f[j] - st[j].x) * st[j].y, sum[j].y);
        }
      }
    if (S > 1) {
      float2* r = red + turn * buffer;
      turn ^= 1;
#pragma unroll
      for (int j = 0; j < W; ++j) r[(s * W + j) * 32 + lane] = sum[j];
      __syncthreads();
#pragma unroll
      for (int j = 0; j < W; ++j) {
        sum[j] = make_float2(0.f, 0.f);
        for (int i = 0; i < S; ++i) {
          const float2 p = r[(i * W + j) * 32 + lane];
          sum[j].x += p.x;
          sum[j].y += p.y;
        }
      }
    }
    float pw[kChanCpt], pb[kChanCpt];
    T* dx = static_cast<T*>(a.y) + at;
#pragma unroll
    for (int k = 0; k < kChanCpt; ++k, advance(dx, step)) {
      pw[k] = pb[k] = 0.f;
      if (k < mine) {
        const float w = lds1(wsm + k * S + s);
        float f[W], g[W];
        renew(x[k].v);
        renew(d[k].v);
        x[k].get(f);
        d[k].get(g);
#pragma unroll
        for (int j = 0; j < W; ++j) {
          const float xh = (f[j] - st[j].x) * st[j].y;
          pw[k] = fmaf(g[j], xh, pw[k]);
          pb[k] += g[j];
          f[j] = st[j].y * (fmaf(g[j], w, -sum[j].x * rc) - xh * (sum[j].y * rc));
        }
        if (in) Word<T, W>::store(dx, f);
      }
    }
    if (a.part != nullptr) {
      dw += transpose_sum(pw, lane);
      db += transpose_sum(pb, lane);
    }
  }
  if (a.part == nullptr) return;
  // the CTA's P tiles, in order, then one partial per CTA
  __syncthreads();
  float2* acc = ln_sm + a.C;  // [P][S][32]
  acc[(threadIdx.z * S + s) * 32 + lane] = make_float2(dw, db);
  __syncthreads();
  if (threadIdx.z == 0 && lane < mine) {
    float2 t = acc[s * 32 + lane];
    for (int p = 1; p < P; ++p) {
      t.x += acc[(p * S + s) * 32 + lane].x;
      t.y += acc[(p * S + s) * 32 + lane].y;
    }
    float* part = a.part + (long long)blockIdx.x * 2 * a.C;
    part[lane * S + s] = t.x;
    part[a.C + lane * S + s] = t.y;
  }
}

// ------------------------------ host side ------------------------------
// How a call runs.  kAny covers what does not fit into registers.
enum LnForm { kRows, kChan, kAny };
struct LnPlan {
  LnForm form;
  int vec;      // kRows: 16-byte vectors; kChan: two 16-bit tokens per word
  int ept;      // kRows: elements per thread
  int G;        // kRows: threads per row
  int threads;  // kRows: of a CTA
  int S, P;     // kChan: warps per tile, tiles per CTA
  long long units;  // CTA-sized pieces of work
};

// Rows: as few threads per row as hold it at 8 elements each (2 vectors of fp32, 1 of
// 16-bit data), more elements only past the largest CTA.  Backward threads also hold
// their columns' weight-grad sums, so their CTAs and elements are fewer.
LnPlan plan_rows(long long tokens, int C, bool vec, bool bwd) {
  LnPlan p{};
  const int most = bwd ? 512 : 1024;
  p.vec = vec;
  for (p.ept = 8; p.ept <= (bwd ? 16 : 32); p.ept *= 2) {
    const int need = (C + p.ept - 1) / p.ept;
    if (!vec && p.ept > 8) break;  // single elements take a register each
    if (need > most) continue;
    p.G = 1;
    while (p.G < need && p.G < 32) p.G *= 2;
    if (need > 32) p.G = (need + 31) / 32 * 32;
    p.threads = p.G <= 32 ? 256 : std::max(1, 256 / p.G) * p.G;
    p.form = kRows;
    const int rows = p.threads / p.G;
    p.units = (tokens + rows - 1) / rows;
    return p;
  }
  p.form = kAny;
  return p;
}

// Channels first: 32 channels per thread, up to 32 warps forward (1024 channels), 16
// backward (512: its threads hold x and dy).
LnPlan plan_chan(long long outer, long long inner, int C, bool pair, bool bwd) {
  LnPlan p{};
  p.S = (C + kChanCpt - 1) / kChanCpt;
  if (p.S > (bwd ? 16 : 32)) {
    p.form = kAny;
    return p;
  }
  p.form = kChan;
  p.vec = pair;
  p.P = std::max(1, 4 / p.S);
  const long long w = pair ? 64 : 32;
  p.units = (outer * ((inner + w - 1) / w) + p.P - 1) / p.P;
  return p;
}

bool aligned_to(const LnArgs& a, size_t n) {
  return ((reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.y) | reinterpret_cast<uintptr_t>(a.dy)) %
          n) == 0;
}

template <typename T>
LnPlan plan_ln(const LnArgs& a, bool bwd) {
  if (a.inner == 1) return plan_rows(a.tokens, a.C, a.C % (16 / sizeof(T)) == 0 && aligned_to(a, 16), bwd);
  return plan_chan(a.outer, a.inner, a.C, sizeof(T) == 2 && a.inner % 2 == 0 && aligned_to(a, 4), bwd);
}

// Most weight-grad partials that a call makes: one per CTA of the backward kernel, four
// CTAs per SM; at least four tokens each, so that the partials stay small beside the data.
int dw_parts(long long tokens) { return (int)std::max(1LL, std::min((long long)kSms * 4, (tokens + 3) / 4)); }

template <typename T, int VEC, int EPT, int R, int THREADS>
int launch_rows_fwd_as(const LnArgs& a, const LnPlan& p, cudaStream_t s) {
  // as many CTAs as the registers of the launch bounds let reside: 768 or 1024 threads
  const long long cap = kSms * (long long)((R > 1 ? 768 : 1024) / p.threads);
  ln_rows_fwd_kernel<T, VEC, EPT, R, THREADS>
      <<<(unsigned)std::min((p.units + R - 1) / R, cap), p.threads, 0, s>>>(a, p.G);
  return record_launch();
}
template <typename T, int VEC, int EPT>
int launch_rows_fwd(const LnArgs& a, const LnPlan& p, cudaStream_t s) {
  if constexpr (EPT == 8) {
    // four rows in flight per thread once every SM has that much to do
    if (p.threads <= 256 && p.units >= kSms * 32) return launch_rows_fwd_as<T, VEC, EPT, 4, 256>(a, p, s);
    if (p.threads <= 256) return launch_rows_fwd_as<T, VEC, EPT, 1, 256>(a, p, s);
  }
  return launch_rows_fwd_as<T, VEC, EPT, 1, 1024>(a, p, s);
}
template <typename T, int VEC, int EPT, int R, int THREADS>
int launch_rows_bwd_as(const LnArgs& a, const LnPlan& p, int parts, cudaStream_t s) {
  auto kern = ln_rows_bwd_kernel<T, VEC, EPT, R, THREADS>;
  const int slots = p.G < 32 ? p.threads / 32 : p.threads / p.G;
  const size_t smem = a.part != nullptr ? (size_t)slots * 2 * a.C * sizeof(float) : 0;
  const int st = ensure_smem(kern, smem);
  if (st != MEDNEXT_OK) return st;
  kern<<<parts, p.threads, smem, s>>>(a, p.G);
  return record_launch();
}
template <typename T, int VEC, int EPT>
int launch_rows_bwd(const LnArgs& a, const LnPlan& p, int parts, cudaStream_t s) {
  if constexpr (EPT == 8) {
    if (p.threads <= 256 && p.units >= 2 * parts) return launch_rows_bwd_as<T, VEC, EPT, 2, 256>(a, p, parts, s);
    if (p.threads <= 256) return launch_rows_bwd_as<T, VEC, EPT, 1, 256>(a, p, parts, s);
  }
  return launch_rows_bwd_as<T, VEC, EPT, 1, 512>(a, p, parts, s);
}

size_t chan_smem(const LnPlan& p, int C) {
  return ((size_t)C + 2 * (size_t)p.P * p.S * (p.vec ? 2 : 1) * 32) * sizeof(float2);
}
template <typename T, int W, int THREADS>
int launch_chan_fwd_as(const LnArgs& a, const LnPlan& p, cudaStream_t s) {
  auto kern = ln_chan_fwd_kernel<T, W, THREADS>;
  const size_t smem = chan_smem(p, a.C);
  const int st = ensure_smem(kern, smem);
  if (st != MEDNEXT_OK) return st;
  const long long cap = kSms * (long long)std::max(1, 24 / (p.S * p.P));  // resident: 24 warps
  kern<<<(unsigned)std::min(p.units, cap), dim3(32, p.S, p.P), smem, s>>>(a);
  return record_launch();
}
template <typename T, int W>
int launch_chan_fwd(const LnArgs& a, const LnPlan& p, cudaStream_t s) {
  return p.S <= 8 ? launch_chan_fwd_as<T, W, 256>(a, p, s) : launch_chan_fwd_as<T, W, 1024>(a, p, s);
}
template <typename T, int W, int THREADS>
int launch_chan_bwd_as(const LnArgs& a, const LnPlan& p, int parts, cudaStream_t s) {
  auto kern = ln_chan_bwd_kernel<T, W, THREADS>;
  const size_t smem = chan_smem(p, a.C);
  const int st = ensure_smem(kern, smem);
  if (st != MEDNEXT_OK) return st;
  kern<<<parts, dim3(32, p.S, p.P), smem, s>>>(a);
  return record_launch();
}
template <typename T, int W>
int launch_chan_bwd(const LnArgs& a, const LnPlan& p, int parts, cudaStream_t s) {
  return p.S <= 8 ? launch_chan_bwd_as<T, W, 256>(a, p, parts, s) : launch_chan_bwd_as<T, W, 512>(a, p, parts, s);
}

template <typename T>
int ln_fwd(const LnArgs& a, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  const LnPlan p = plan_ln<T>(a, false);
  if (p.form == kRows) {
    if (p.ept == 8) return p.vec ? launch_rows_fwd<T, V, 8>(a, p, s) : launch_rows_fwd<T, 1, 8>(a, p, s);
    if (p.ept == 16) return launch_rows_fwd<T, V, 16>(a, p, s);
    return launch_rows_fwd<T, V, 32>(a, p, s);
  }
  if (p.form == kChan) {
    if constexpr (sizeof(T) == 2)
      if (p.vec) return launch_chan_fwd<T, 2>(a, p, s);
    return launch_chan_fwd<T, 1>(a, p, s);
  }
  if (a.inner == 1) {
    ln_rows_any_fwd_kernel<T><<<(unsigned)std::min<long long>(a.tokens, kSms * 32), 256, 0, s>>>(a);
  } else {
    const long long tiles = a.outer * ((a.inner + 31) / 32);
    ln_chan_any_fwd_kernel<T><<<(unsigned)std::min<long long>(tiles, kSms * 32), 256, 0, s>>>(a);
  }
  return record_launch();
}

template <typename T>
int ln_bwd(const LnArgs& a, void* dw, void* db, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  const LnPlan p = plan_ln<T>(a, true);
  // one CTA per resident slot (the launch bounds leave 512 threads), one partial per CTA
  const int warps = p.form == kRows ? p.threads / 32 : p.S * p.P;
  const long long slots = (long long)kSms * std::max(1, 16 / std::max(1, warps));
  int st, parts = (int)std::min<long long>(std::min<long long>(dw_parts(a.tokens), slots), std::max(1LL, p.units));
  if (p.form == kRows) {
    if (p.ept == 8)
      st = p.vec ? launch_rows_bwd<T, V, 8>(a, p, parts, s) : launch_rows_bwd<T, 1, 8>(a, p, parts, s);
    else
      st = launch_rows_bwd<T, V, 16>(a, p, parts, s);
  } else if (p.form == kChan) {
    if constexpr (sizeof(T) == 2)
      st = p.vec ? launch_chan_bwd<T, 2>(a, p, parts, s) : launch_chan_bwd<T, 1>(a, p, parts, s);
    else
      st = launch_chan_bwd<T, 1>(a, p, parts, s);
  } else {
    // enough CTAs for the GPU over the columns and the parts
    const long long cols = a.inner == 1 ? (a.C + 31) / 32 : a.C;
    parts = (int)std::min<long long>(dw_parts(a.tokens), std::max(1LL, (long long)kSms * 8 / cols));
    if (a.inner == 1) {
      ln_rows_any_dx_kernel<T><<<(unsigned)std::min<long long>(a.tokens, kSms * 32), 256, 0, s>>>(a);
    } else {
      const long long tiles = a.outer * ((a.inner + 31) / 32);
      ln_chan_any_dx_kernel<T><<<(unsigned)std::min<long long>(tiles, kSms * 32), 256, 0, s>>>(a);
    }
    st = record_launch();
    if (st != MEDNEXT_OK || a.part == nullptr) return st;
    if (a.inner == 1)
      ln_rows_any_dw_kernel<T><<<dim3((a.C + 31) / 32, parts), 256, 0, s>>>(a, parts);
    else
      ln_chan_any_dw_kernel<T><<<dim3(a.C, parts), 256, 0, s>>>(a, parts);
    st = record_launch();
  }
  if (st != MEDNEXT_OK || a.part == nullptr) return st;
  ln_fold_kernel<<<(a.C + 31) / 32, 1024, 0, s>>>(a.part, parts, a.C, dw, db, a.pdt);
  return record_launch();
}

// Everything that both directions check.  Token and channel counts below 2^31 keep the
// kernels' channel indexes in 32 bits; element offsets are 64-bit.
int ln_check(int64_t outer, int64_t c, int64_t inner, int dtype, int param_dtype) {
  if (dtype != MEDNEXT_FLOAT32 && dtype != MEDNEXT_BFLOAT16 && dtype != MEDNEXT_FLOAT16) return MEDNEXT_ERR_BAD_DTYPE;
  if (param_dtype != MEDNEXT_FLOAT32 && param_dtype != dtype) return MEDNEXT_ERR_BAD_DTYPE;
  if (outer < 0 || inner < 0 || c <= 0 || c > ((int64_t)1 << 24)) return MEDNEXT_ERR_BAD_SHAPE;
  const int64_t lim = (int64_t)1 << 40;  // tokens, and elements
  if (outer >= lim || inner >= lim) return MEDNEXT_ERR_BAD_SHAPE;
  if (outer > 0 && inner > 0 && (inner > lim / outer || outer * inner > lim / c)) return MEDNEXT_ERR_BAD_SHAPE;
  return MEDNEXT_OK;
}

bool misaligned(const void* p, int dtype) { return reinterpret_cast<uintptr_t>(p) % elem_size(dtype) != 0; }

}  // namespace
}  // namespace mednext

using namespace mednext;

int mednext_ln_fwd(const void* x, const void* weight, const void* bias, void* y, float* stats, int64_t outer,
                   int64_t c, int64_t inner, float eps, int dtype, int param_dtype, mednext_stream_t stream) {
  const int st = ln_check(outer, c, inner, dtype, param_dtype);
  if (st != MEDNEXT_OK) return st;
  if (!(eps > 0.f) || !(eps < INFINITY)) return MEDNEXT_ERR_BAD_VALUE;
  if (outer * inner == 0) return MEDNEXT_OK;
  if (x == nullptr || y == nullptr) return MEDNEXT_ERR_NULL_POINTER;
  if (misaligned(x, dtype) || misaligned(y, dtype) || misaligned(weight, param_dtype) ||
      misaligned(bias, param_dtype) || (reinterpret_cast<uintptr_t>(stats) & 7))
    return MEDNEXT_ERR_ALIGNMENT;
  LnArgs a{};
  a.x = x; a.w = weight; a.b = bias; a.y = y;
  a.stats = reinterpret_cast<float2*>(stats);
  a.outer = outer; a.inner = inner; a.tokens = outer * inner; a.C = (int)c;
  a.pdt = param_dtype; a.eps = eps;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  switch (dtype) {
    case MEDNEXT_FLOAT32: return ln_fwd<float>(a, s);
    case MEDNEXT_BFLOAT16: return ln_fwd<__nv_bfloat16>(a, s);
    default: return ln_fwd<__half>(a, s);
  }
}

size_t mednext_ln_bwd_workspace_size(int64_t outer, int64_t c, int64_t inner, int dtype) {
  if (ln_check(outer, c, inner, dtype, MEDNEXT_FLOAT32) != MEDNEXT_OK || outer * inner == 0) return 0;
  return (size_t)dw_parts(outer * inner) * 2 * (size_t)c * sizeof(float);
}

int mednext_ln_bwd(const void* dy, const void* x, const float* stats, const void* weight, void* dx, void* dweight,
                   void* dbias, void* workspace, size_t workspace_bytes, int64_t outer, int64_t c, int64_t inner,
                   int dtype, int param_dtype, mednext_stream_t stream) {
  const int st = ln_check(outer, c, inner, dtype, param_dtype);
  if (st != MEDNEXT_OK) return st;
  if (misaligned(dweight, param_dtype) || misaligned(dbias, param_dtype)) return MEDNEXT_ERR_ALIGNMENT;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const bool params = dweight != nullptr || dbias != nullptr;
  if (outer * inner == 0) {
    if (!params) return MEDNEXT_OK;
    ln_fold_kernel<<<(unsigned)((c + 31) / 32), 1024, 0, s>>>(nullptr, 0, (int)c, dweight, dbias, param_dtype);
    return record_launch();
  }
  if (dy == nullptr || x == nullptr || stats == nullptr || dx == nullptr) return MEDNEXT_ERR_NULL_POINTER;
  if (misaligned(dy, dtype) || misaligned(x, dtype) || misaligned(dx, dtype) || misaligned(weight, param_dtype) ||
      (reinterpret_cast<uintptr_t>(stats) & 7))
    return MEDNEXT_ERR_ALIGNMENT;
  if (params && (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 15) ||
                 workspace_bytes < mednext_ln_bwd_workspace_size(outer, c, inner, dtype)))
    return MEDNEXT_ERR_WORKSPACE;
  LnArgs a{};
  a.x = x; a.dy = dy; a.w = weight; a.y = dx;
  a.stats = reinterpret_cast<float2*>(const_cast<float*>(stats));
  a.part = params ? static_cast<float*>(workspace) : nullptr;
  a.outer = outer; a.inner = inner; a.tokens = outer * inner; a.C = (int)c;
  a.pdt = param_dtype;
  switch (dtype) {
    case MEDNEXT_FLOAT32: return ln_bwd<float>(a, dweight, dbias, s);
    case MEDNEXT_BFLOAT16: return ln_bwd<__nv_bfloat16>(a, dweight, dbias, s);
    default: return ln_bwd<__half>(a, dweight, dbias, s);
  }
}
