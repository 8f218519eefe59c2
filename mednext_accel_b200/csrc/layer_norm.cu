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

// dw, db = the partials' sums, in the order of the parts: 8 warps take every eighth
// part of 32 columns, then one adds the 8 sums.  parts = 0 writes zeros (no tokens).
__global__ void __launch_bounds__(256) ln_fold_kernel(const float* __restrict__ part, int parts, int C, void* dw,
                                                      void* db, int pdt) {
  __shared__ double red[2][8][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  double s0 = 0.0, s1 = 0.0;
  if (c < C)
    for (int p = warp; p < parts; p += 8) {
      s0 += (double)part[((long long)p * 2) * C + c];
      s1 += (double)part[((long long)p * 2 + 1) * C + c];
    }
  red[0][warp][lane] = s0;
  red[1][warp][lane] = s1;
  __syncthreads();
  if (warp == 0 && c < C) {
    for (int w = 1; w < 8; ++w) {
      s0 += red[0][w][lane];
      s1 += red[1][w][lane];
    }
    store_param(dw, pdt, c, s0);
    store_param(db, pdt, c, s1);
  }
}

// ------------------------------ host side ------------------------------
// Parts of the tokens that the weight-grad partials are taken over: enough CTAs for
// the GPU, at least 64 tokens each.
int dw_parts(long long tokens, int C, long long inner) {
  const long long cols = inner == 1 ? (C + 31) / 32 : C;
  const long long want = std::max(1LL, (long long)kSms * 8 / cols);
  return (int)std::max(1LL, std::min(want, (tokens + 63) / 64));
}

template <typename T>
int ln_fwd(const LnArgs& a, cudaStream_t s) {
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
  if (a.inner == 1) {
    ln_rows_any_dx_kernel<T><<<(unsigned)std::min<long long>(a.tokens, kSms * 32), 256, 0, s>>>(a);
  } else {
    const long long tiles = a.outer * ((a.inner + 31) / 32);
    ln_chan_any_dx_kernel<T><<<(unsigned)std::min<long long>(tiles, kSms * 32), 256, 0, s>>>(a);
  }
  int st = record_launch();
  if (st != MEDNEXT_OK || a.part == nullptr) return st;
  const int parts = dw_parts(a.tokens, a.C, a.inner);
  if (a.inner == 1)
    ln_rows_any_dw_kernel<T><<<dim3((a.C + 31) / 32, parts), 256, 0, s>>>(a, parts);
  else
    ln_chan_any_dw_kernel<T><<<dim3(a.C, parts), 256, 0, s>>>(a, parts);
  st = record_launch();
  if (st != MEDNEXT_OK) return st;
  ln_fold_kernel<<<(a.C + 31) / 32, 256, 0, s>>>(a.part, parts, a.C, dw, db, a.pdt);
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
  return (size_t)dw_parts(outer * inner, (int)c, inner) * 2 * (size_t)c * sizeof(float);
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
    ln_fold_kernel<<<(unsigned)((c + 31) / 32), 256, 0, s>>>(nullptr, 0, (int)c, dweight, dbias, param_dtype);
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
