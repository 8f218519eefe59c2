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
constexpr int kChanMost = 16384;  // channels of the channels-first form

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
// Past 8192 columns, or 2048 where rows are read by single elements.  One CTA per row at a time; the
// row is read again for each pass (from L1 / L2), an element at a time, which bounds it: 5000 x 4095 bf16 74 us
// forward, 111 us backward, 1.1 TB/s of what the call has to move.
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

__device__ __forceinline__ void store_param(void* p, int dtype, int i, double v) {
  if (p == nullptr) return;
  if (dtype == MEDNEXT_FLOAT32) static_cast<float*>(p)[i] = (float)v;
  else if (dtype == MEDNEXT_BFLOAT16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn((float)v);
  else static_cast<__half*>(p)[i] = __float2half_rn((float)v);
}

// dw, db = the partials' sums in a fixed order: 32 warps take every 32nd part of 32
// columns, then one adds the 32 sums.  parts = 0 writes zeros (no tokens).  part is plain memory
// (not __restrict__, which would allow read-only loads): it is launched while part is written.
__global__ void __launch_bounds__(1024) ln_fold_kernel(const float* part, int parts, int C, void* dw, void* db, int pdt) {
  __shared__ double red[2][32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  double s0 = 0.0, s1 = 0.0;
  grid_dependency_wait();
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

// ------------------------------ packed arithmetic ------------------------------
// All of the register kernels below work on pairs (fp32 x 2 instructions) of values that
// stay packed in their own type until they are used: these kernels are bound by
// instruction issue as soon as their loads are wide, so an element's instructions count.
// centered() subtracts a mean from the packed pair itself, by a mixed-precision FMA with 1
// for the 16-bit types: the same bits as widening and subtracting, without the widening.
template <typename T>
struct Pack {  // 16-bit types: two elements per word
  using Word = uint32_t;
  static __device__ __forceinline__ float2 value(uint32_t w) { return unpack2<T>(w); }
  static __device__ __forceinline__ float2 plus(uint32_t w, float2 add) {
    return make_float2(mix_fma<T>((uint16_t)(w & 0xffffu), one16<T>(), add.x),
                       mix_fma<T>((uint16_t)(w >> 16), one16<T>(), add.y));
  }
  static __device__ __forceinline__ uint32_t make(float2 v) { return pack2<T>(v); }
};
template <>
struct Pack<float> {
  using Word = float2;
  static __device__ __forceinline__ float2 value(float2 w) { return w; }
  static __device__ __forceinline__ float2 plus(float2 w, float2 add) { return __fadd2_rn(w, add); }
  static __device__ __forceinline__ float2 make(float2 v) { return v; }
};
// Two 16-bit elements in a register each, as single-element loads leave them: packing them
// would wait for each pair before the next load.
struct Halves {
  uint16_t a, b;
};
template <typename T>
struct Apart {
  using Word = Halves;
  static __device__ __forceinline__ float2 value(Halves w) {
    return make_float2(to_acc<T>(reinterpret_cast<const T&>(w.a)), to_acc<T>(reinterpret_cast<const T&>(w.b)));
  }
  static __device__ __forceinline__ float2 plus(Halves w, float2 add) {
    return make_float2(mix_fma<T>(w.a, one16<T>(), add.x), mix_fma<T>(w.b, one16<T>(), add.y));
  }
};
template <>
struct Apart<float> : Pack<float> {};
template <typename T, bool SINGLE>
struct PackFor : Pack<T> {};
template <typename T>
struct PackFor<T, true> : Apart<T> {};

// Makes the compiler take the packed words as new values: it unpacks them again (one
// instruction for a bf16) instead of keeping the unpacked copies in registers.
__device__ __forceinline__ void renew(uint32_t& v) { asm volatile("" : "+r"(v)); }
__device__ __forceinline__ void renew(float2&) {}
__device__ __forceinline__ void renew(Halves& v) { asm volatile("" : "+h"(v.a), "+h"(v.b)); }

// A 16-byte load that is issued where it is written (zeros if not ok): left to itself the
// compiler sinks the loads for the next rows behind the work on these.
__device__ __forceinline__ uint4 load_here(const void* p, bool ok) {
  uint4 q;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.u32 p, %5, 0;\n\t"
      "mov.u32 %0, 0;\n\tmov.u32 %1, 0;\n\tmov.u32 %2, 0;\n\tmov.u32 %3, 0;\n\t"
      "@p ld.global.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
      : "=&r"(q.x), "=&r"(q.y), "=&r"(q.z), "=&r"(q.w)
      : "l"(p), "r"((uint32_t)ok));
  return q;
}

// ------------------------------ rows held in registers ------------------------------
// G threads hold a row, EPT elements each, in words of VEC elements (16 bytes; 4 bytes or
// single elements where rows do not start on 16), word v of thread gl beginning at column
// (v G + gl) VEC.  G <= 32 is a power of two and its sums are shuffles; wider rows take
// whole warps, which add through shared memory, one barrier of the group per sum, R rows at
// once.
template <typename T, int VEC, int EPT>
struct RowFrag {
  using P = PackFor<T, VEC == 1>;
  static constexpr int kChunk = VEC == 1 ? 2 : VEC;  // elements handled together
  static constexpr int kChunks = EPT / kChunk, kPairs = kChunk / 2;
  typename P::Word w[EPT / 2];
  static __device__ __forceinline__ int col(int j, int e, int gl, int G) {  // of element e of chunk j
    return VEC == 1 ? (2 * j + e) * G + gl : (j * G + gl) * VEC + e;
  }
  __device__ __forceinline__ void load(const T* row, int gl, int G, int C, bool in) {
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
      if constexpr (VEC == 1) {
        const int c0 = col(j, 0, gl, G), c1 = col(j, 1, gl, G);
        const T a = in && c0 < C ? row[c0] : from_acc<T>(0.f), b = in && c1 < C ? row[c1] : from_acc<T>(0.f);
        if constexpr (sizeof(T) == 4) w[j] = make_float2(a, b);
        else w[j] = Halves{reinterpret_cast<const uint16_t&>(a), reinterpret_cast<const uint16_t&>(b)};
      } else {
        const int c = col(j, 0, gl, G);
        const bool ok = in && c < C;
        if constexpr (sizeof(T) * VEC == 16) {
          const uint4 q = load_here(row + c, ok);
          if constexpr (sizeof(T) == 4) {
            w[2 * j] = make_float2(__uint_as_float(q.x), __uint_as_float(q.y));
            w[2 * j + 1] = make_float2(__uint_as_float(q.z), __uint_as_float(q.w));
          } else {
            w[4 * j] = q.x; w[4 * j + 1] = q.y; w[4 * j + 2] = q.z; w[4 * j + 3] = q.w;
          }
        } else {
          w[j] = ok ? *reinterpret_cast<const uint32_t*>(row + c) : 0u;
        }
      }
    }
  }
  __device__ __forceinline__ void again() {
#pragma unroll
    for (int i = 0; i < EPT / 2; ++i) renew(w[i]);
  }
  // f: the chunk's pairs
  static __device__ __forceinline__ void store(T* row, int j, int gl, int G, int C, const float2* f) {
    const int c = col(j, 0, gl, G);
    if constexpr (VEC == 1) {
      if (c < C) row[c] = from_acc<T>(f[0].x);
      if (c + G < C) row[c + G] = from_acc<T>(f[0].y);
    } else if constexpr (sizeof(T) * VEC == 16) {
      if (c >= C) return;
      if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(row + c) = make_float4(f[0].x, f[0].y, f[1].x, f[1].y);
      else *reinterpret_cast<uint4*>(row + c) = make_uint4(P::make(f[0]), P::make(f[1]), P::make(f[2]), P::make(f[3]));
    } else {
      if (c < C) *reinterpret_cast<uint32_t*>(row + c) = P::make(f[0]);
    }
  }
};

// A parameter vector for the fragments: in registers up to 16 elements per thread, else in
// shared memory (EPT * G floats), where 8-element words are split into two planes of
// four so that the lanes of a 16-byte load lie side by side.
template <typename T, int VEC, int EPT>
struct RowParam {
  using Frag = RowFrag<T, VEC, EPT>;
  static constexpr bool kRegs = EPT <= 16;
  float2 r[kRegs ? EPT / 2 : 1];
  const float* sm;
  static size_t smem_bytes(int G) { return kRegs ? 0 : (size_t)EPT * G * sizeof(float); }
  static __device__ __forceinline__ int place(int c, int G) {
    if constexpr (VEC == 8) return (((c >> 3) / G * 2 + ((c >> 2) & 1)) * G + (c >> 3) % G) * 4 + (c & 3);
    else return c;
  }
  template <typename F>
  __device__ __forceinline__ void regs(F at, int gl, int G, int C) {
#pragma unroll
    for (int i = 0; i < EPT / 2; ++i) {
      const int j = i / Frag::kPairs, e = i % Frag::kPairs * 2;
      const int c0 = Frag::col(j, e, gl, G), c1 = Frag::col(j, e + 1, gl, G);
      r[i] = make_float2(c0 < C ? at(c0) : 0.f, c1 < C ? at(c1) : 0.f);
    }
  }
  // every thread of the CTA calls this; a barrier follows where shared memory is used
  __device__ __forceinline__ void fill(const void* p, int dtype, float none, float* smem, int gl, int G, int C) {
    sm = smem;
    if constexpr (kRegs) {
      // the type is told apart once, so that the loads of one vector are in flight together
      if (p == nullptr) regs([=](int) { return none; }, gl, G, C);
      else if (dtype == MEDNEXT_FLOAT32) regs([=](int c) { return static_cast<const float*>(p)[c]; }, gl, G, C);
      else regs([=](int c) { return to_acc<T>(static_cast<const T*>(p)[c]); }, gl, G, C);
    } else {
      for (int c = threadIdx.x; c < EPT * G; c += blockDim.x)
        smem[place(c, G)] = c < C ? load_param(p, dtype, c, none) : 0.f;
    }
  }
  __device__ __forceinline__ void get(int j, int gl, int G, float2* f) const {  // the chunk's pairs
    if constexpr (kRegs) {
#pragma unroll
      for (int i = 0; i < Frag::kPairs; ++i) f[i] = r[j * Frag::kPairs + i];
    } else if constexpr (VEC == 8) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float4 q = *reinterpret_cast<const float4*>(sm + ((2 * j + h) * G + gl) * 4);
        f[2 * h] = make_float2(q.x, q.y);
        f[2 * h + 1] = make_float2(q.z, q.w);
      }
    } else if constexpr (VEC == 4) {
      const float4 q = *reinterpret_cast<const float4*>(sm + (j * G + gl) * 4);
      f[0] = make_float2(q.x, q.y);
      f[1] = make_float2(q.z, q.w);
    } else if constexpr (VEC == 2) {
      f[0] = *reinterpret_cast<const float2*>(sm + (j * G + gl) * 2);
    } else {
      f[0] = make_float2(sm[Frag::col(j, 0, gl, G)], sm[Frag::col(j, 1, gl, G)]);
    }
  }
};

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
  // the groups of a CTA go their own ways
  asm volatile("bar.sync %0, %1;" ::"r"((int)threadIdx.x / G + 1), "r"(G) : "memory");
  const int w0 = (threadIdx.x / G) * (G >> 5), w1 = w0 + (G >> 5);
#pragma unroll
  for (int n = 0; n < N; ++n) v[n] = 0.f;
  for (int w = w0; w < w1; ++w) {
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] += r[n * 32 + w];
  }
}

constexpr int kRowThreads = 256;

// Rows of 16-bit data of odd width start at any element, and a warp's single elements are 64-byte
// pieces off their sectors: 1.4 TB/s whatever the elements per thread (8, 16 or 32).  A CTA's rows are one
// block of memory, though: with enough of them it goes through shared memory in 16-byte words, and
// the threads take their elements from there (RowBlock).
template <typename T, int VEC, int R>
constexpr bool kBlockRows = VEC == 1 && sizeof(T) == 2 && R > 1;
// The next rows are on their way while a group works on its rows: a group is one or a few
// warps, too few per SM to hide the loads' latency by their number.  Bound by HBM on long
// rows (4096 x 4096 fp32: 25 us, 5.4 TB/s), by latency and start-up on few or short ones
// (16384 x 1024 bf16: 17.8 us, 3.8 TB/s); single-element words by instruction issue
// (30000 x 777 bf16: 50 us, 1.9 TB/s; without RowBlock 62).
template <typename T, int VEC, int EPT, int R>
__global__ void __launch_bounds__(kRowThreads, 2) ln_rows_fwd_kernel(LnArgs a, int G) {
  using Frag = RowFrag<T, VEC, EPT>;
  using P = typename Frag::P;
  extern __shared__ __align__(16) float ln_sm[];
  __shared__ float red[2 * R * 32];
  int turn = 0;
  const int groups = blockDim.x / G, gi = threadIdx.x / G, gl = threadIdx.x - gi * G;
  const float rc = 1.f / (float)a.C;
  const long long stride = (long long)gridDim.x * groups * R;
  Frag next[R];
  // (block rows: [2] blocks of x, a block of y)
  constexpr bool kBlock = kBlockRows<T, VEC, R>;
  uint8_t* block = reinterpret_cast<uint8_t*>(ln_sm);
  const int bytes = block_bytes<T>(groups * R, a.C);
  int buf = 0;
  const auto of_block = [&](long long base) { return (int)min((long long)groups * R, a.tokens - base) * a.C; };
  const auto load = [&](long long base) {
    if constexpr (kBlock) {
      if (base < a.tokens) RowBlock<T>::fetch(block + buf * bytes, static_cast<const T*>(a.x) + base * a.C, of_block(base));
      return;
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long t = base + r * groups + gi;
      next[r].load(static_cast<const T*>(a.x) + t * a.C, gl, G, a.C, t < a.tokens);
    }
  };
  load((long long)blockIdx.x * groups * R);
  RowParam<T, VEC, EPT> w, b;
  w.fill(a.w, a.pdt, 1.f, ln_sm, gl, G, a.C);
  b.fill(a.b, a.pdt, 0.f, ln_sm + EPT * G, gl, G, a.C);
  if (!w.kRegs) __syncthreads();
  for (long long base = (long long)blockIdx.x * groups * R; base < a.tokens; base += stride) {
    Frag x[R];
    float s[R];
    if constexpr (kBlock) {
      RowBlock<T>::arrived();
      __syncthreads();  // the block is there, the last block of y has been stored
      const T* xs = RowBlock<T>::first(block + buf * bytes, static_cast<const T*>(a.x) + base * a.C);
#pragma unroll
      for (int r = 0; r < R; ++r)
        x[r].load(xs + (r * groups + gi) * a.C, gl, G, a.C, base + r * groups + gi < a.tokens);
      buf ^= 1;
    } else {
#pragma unroll
      for (int r = 0; r < R; ++r) x[r] = next[r];
    }
    if (base + stride < a.tokens) load(base + stride);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float2 sum = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < EPT / 2; ++i) sum = P::plus(x[r].w[i], sum);
      s[r] = sum.x + sum.y;
    }
    group_sum<R>(s, G, red, turn);
    float2 nm[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      nm[r] = f2(-s[r] * rc);
      x[r].again();
      float2 sq = make_float2(0.f, 0.f);
#pragma unroll
      for (int j = 0; j < Frag::kChunks; ++j) {
        if (VEC > 1 && Frag::col(j, 0, gl, G) >= a.C) continue;
#pragma unroll
        for (int i = 0; i < Frag::kPairs; ++i) {
          float2 d = P::plus(x[r].w[j * Frag::kPairs + i], nm[r]);
          if (VEC == 1) {
            if (Frag::col(j, 0, gl, G) >= a.C) d.x = 0.f;
            if (Frag::col(j, 1, gl, G) >= a.C) d.y = 0.f;
          }
          sq = __ffma2_rn(d, d, sq);
        }
      }
      s[r] = sq.x + sq.y;
    }
    group_sum<R>(s, G, red, turn);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long t = base + r * groups + gi;
      if (t >= a.tokens) continue;
      x[r].again();
      const float rstd = rsqrtf(s[r] * rc + a.eps);
      T* y = static_cast<T*>(a.y) + t * a.C;
      if constexpr (kBlock)
        y = RowBlock<T>::first(block + 2 * bytes, static_cast<T*>(a.y) + base * a.C) + (r * groups + gi) * a.C;
#pragma unroll
      for (int j = 0; j < Frag::kChunks; ++j) {
        float2 f[Frag::kPairs], pw[Frag::kPairs], pb[Frag::kPairs];
        w.get(j, gl, G, pw);
        b.get(j, gl, G, pb);
#pragma unroll
        for (int i = 0; i < Frag::kPairs; ++i)
          f[i] = __ffma2_rn(__fmul2_rn(P::plus(x[r].w[j * Frag::kPairs + i], nm[r]), f2(rstd)), pw[i], pb[i]);
        Frag::store(y, j, gl, G, a.C, f);
      }
      if (a.stats != nullptr && gl == 0) a.stats[t] = make_float2(-nm[r].x, rstd);
    }
    if constexpr (kBlock) {
      __syncthreads();
      RowBlock<T>::put(static_cast<T*>(a.y) + base * a.C, block + 2 * bytes, of_block(base));
    }
  }
}

// The threads own their columns over all rows of the CTA, so the weight grads are sums
// in registers (4096 x 4096 fp32: 44 us, 4.6 TB/s; 16384 x 1024 bf16: 28 us, 3.6 TB/s,
// the fold of the partials included); the CTA adds its groups' sums through shared memory ([slots][2][C], a
// slot per warp for G <= 32, per group else) and writes one partial per CTA.
template <typename T, int VEC, int EPT, int R>
__global__ void __launch_bounds__(kRowThreads, 2) ln_rows_bwd_kernel(LnArgs a, int G) {
  using Frag = RowFrag<T, VEC, EPT>;
  using P = typename Frag::P;
  extern __shared__ __align__(16) float ln_sm[];
  __shared__ float red[2 * 2 * R * 32];
  grid_dependents_go();
  int turn = 0;
  const int groups = blockDim.x / G, gi = threadIdx.x / G, gl = threadIdx.x - gi * G;
  const float rc = 1.f / (float)a.C;
  constexpr bool kAhead = EPT <= 16;  // 32 elements' sums leave no registers for the next rows
  const long long stride = (long long)gridDim.x * groups * R;
  Frag xn[R], dn[R];
  float2 stn[R];
  // (block rows: [2] blocks of x, of dy, a block of dx)
  constexpr bool kBlock = kBlockRows<T, VEC, R>;
  uint8_t* block = reinterpret_cast<uint8_t*>(ln_sm);
  const int bytes = block_bytes<T>(groups * R, a.C);
  int buf = 0;
  const auto of_block = [&](long long base) { return (int)min((long long)groups * R, a.tokens - base) * a.C; };
  const auto load = [&](long long base) {
    if constexpr (kBlock) {
      if (base < a.tokens) {
        RowBlock<T>::fetch(block + buf * bytes, static_cast<const T*>(a.x) + base * a.C, of_block(base));
        RowBlock<T>::fetch(block + (2 + buf) * bytes, static_cast<const T*>(a.dy) + base * a.C, of_block(base));
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long t = base + r * groups + gi;
      const bool in = t < a.tokens;
      if constexpr (kBlock) {
        stn[r] = in ? a.stats[t] : make_float2(0.f, 0.f);
        continue;
      }
      xn[r].load(static_cast<const T*>(a.x) + t * a.C, gl, G, a.C, in);
      dn[r].load(static_cast<const T*>(a.dy) + t * a.C, gl, G, a.C, in);
      stn[r] = in ? a.stats[t] : make_float2(0.f, 0.f);
    }
  };
  if (kAhead) load((long long)blockIdx.x * groups * R);
  RowParam<T, VEC, EPT> w;
  w.fill(a.w, a.pdt, 1.f, ln_sm, gl, G, a.C);
  if (!w.kRegs) __syncthreads();
  float2 dw[EPT / 2], db[EPT / 2];
#pragma unroll
  for (int i = 0; i < EPT / 2; ++i) dw[i] = db[i] = make_float2(0.f, 0.f);
  for (long long base = (long long)blockIdx.x * groups * R; base < a.tokens; base += stride) {
    Frag x[R], d[R];
    float2 st[R];
    float s[2 * R];
    if (!kAhead) load(base);
    if constexpr (kBlock) {
      RowBlock<T>::arrived();
      __syncthreads();  // the blocks are there, the last block of dx has been stored
      const T* xs = RowBlock<T>::first(block + buf * bytes, static_cast<const T*>(a.x) + base * a.C);
      const T* ds = RowBlock<T>::first(block + (2 + buf) * bytes, static_cast<const T*>(a.dy) + base * a.C);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const bool in = base + r * groups + gi < a.tokens;
        x[r].load(xs + (r * groups + gi) * a.C, gl, G, a.C, in);
        d[r].load(ds + (r * groups + gi) * a.C, gl, G, a.C, in);
        st[r] = stn[r];
      }
      buf ^= 1;
    } else {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        x[r] = xn[r];
        d[r] = dn[r];
        st[r] = stn[r];
      }
    }
    if (kAhead && base + stride < a.tokens) load(base + stride);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float2 s1 = make_float2(0.f, 0.f), s2 = s1;
#pragma unroll
      for (int j = 0; j < Frag::kChunks; ++j) {
        float2 pw[Frag::kPairs];
        w.get(j, gl, G, pw);
#pragma unroll
        for (int i = 0; i < Frag::kPairs; ++i) {
          const int n = j * Frag::kPairs + i;
          const float2 xh = __fmul2_rn(P::plus(x[r].w[n], f2(-st[r].x)), f2(st[r].y));
          const float2 g = P::value(d[r].w[n]), gw = __fmul2_rn(g, pw[i]);
          dw[n] = __ffma2_rn(g, xh, dw[n]);
          db[n] = __fadd2_rn(db[n], g);
          s1 = __fadd2_rn(s1, gw);
          s2 = __ffma2_rn(gw, xh, s2);
        }
      }
      s[2 * r] = s1.x + s1.y;
      s[2 * r + 1] = s2.x + s2.y;
    }
    group_sum<2 * R>(s, G, red, turn);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long t = base + r * groups + gi;
      if (t >= a.tokens) continue;
      x[r].again();
      d[r].again();
      const float2 m1 = f2(-s[2 * r] * rc), m2 = f2(-s[2 * r + 1] * rc);
      T* dx = static_cast<T*>(a.y) + t * a.C;
      if constexpr (kBlock)
        dx = RowBlock<T>::first(block + 4 * bytes, static_cast<T*>(a.y) + base * a.C) + (r * groups + gi) * a.C;
#pragma unroll
      for (int j = 0; j < Frag::kChunks; ++j) {
        float2 f[Frag::kPairs], pw[Frag::kPairs];
        w.get(j, gl, G, pw);
#pragma unroll
        for (int i = 0; i < Frag::kPairs; ++i) {
          const int n = j * Frag::kPairs + i;
          const float2 xh = __fmul2_rn(P::plus(x[r].w[n], f2(-st[r].x)), f2(st[r].y));
          const float2 t1 = __ffma2_rn(P::value(d[r].w[n]), pw[i], m1);
          f[i] = __fmul2_rn(__ffma2_rn(xh, m2, t1), f2(st[r].y));
        }
        Frag::store(dx, j, gl, G, a.C, f);
      }
    }
    if constexpr (kBlock) {
      __syncthreads();
      RowBlock<T>::put(static_cast<T*>(a.y) + base * a.C, block + 4 * bytes, of_block(base));
    }
  }
  if (a.part == nullptr) return;
  // lanes of one warp that hold the same columns, then the CTA's slots, in order
#pragma unroll
  for (int i = 0; i < EPT / 2; ++i)
    for (int o = G; o < 32; o <<= 1) {
      dw[i].x += __shfl_xor_sync(0xffffffffu, dw[i].x, o);
      dw[i].y += __shfl_xor_sync(0xffffffffu, dw[i].y, o);
      db[i].x += __shfl_xor_sync(0xffffffffu, db[i].x, o);
      db[i].y += __shfl_xor_sync(0xffffffffu, db[i].y, o);
    }
  __syncthreads();  // the parameters or blocks in shared memory give way
  const int slot = G < 32 ? threadIdx.x >> 5 : gi, slots = G < 32 ? blockDim.x >> 5 : groups;
  if (G >= 32 || (threadIdx.x & 31) < G) {
#pragma unroll
    for (int i = 0; i < EPT / 2; ++i) {
      const int j = i / Frag::kPairs, e = i % Frag::kPairs * 2;
      const int c0 = Frag::col(j, e, gl, G), c1 = Frag::col(j, e + 1, gl, G);
      float* at = ln_sm + (size_t)(2 * slot) * a.C;
      if (c0 < a.C) {
        at[c0] = dw[i].x;
        at[a.C + c0] = db[i].x;
      }
      if (c1 < a.C) {
        at[c1] = dw[i].y;
        at[a.C + c1] = db[i].y;
      }
    }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < 2 * a.C; c += blockDim.x) {
    float v = 0.f;
    for (int i = 0; i < slots; ++i) v += ln_sm[(size_t)i * 2 * a.C + c];
    a.part[(long long)blockIdx.x * 2 * a.C + c] = v;
  }
}

// ------------------------------ channels first, held in registers ------------------------------
// A lane owns W neighbouring tokens and CPT channels of them; a tile of 32 W tokens takes
// S = ceil(C / CPT) warps, channel k S + s belonging to warp s.  Each load is one coalesced
// segment of a channel's row, and x is read once.  Only two numbers per token cross the
// warps, once per tile.  blockDim = (32, S, P), P tiles per CTA side by side.
//
// W = 4 (8 bytes of 16-bit data) and W = 2 need inner to be a multiple of W and the tensors
// to start on a word; W = 1 takes the rest (odd volumes).  The wider word spends 64-bit
// addresses, parameter loads and predicates on more elements.
//
// A slot is what is computed together: one channel of W tokens (pairs of tokens), or, for
// W = 1, two channels of one token (a pair of channels).
//
// 32 x 128^3 bf16: forward 50 us (5.4 TB/s), backward 82 us (4.9 TB/s), the statistics' 17 MB
// apart.  Issue (about 10 instructions an element forward, 26 with scalar arithmetic and
// 4-byte words: 65 and 111 us) and HBM share the bound; odd volumes (2 x 96 x 33x35x37 fp32: 16.5
// and 36 us) are bound by the single-element words' instructions.
template <typename T, int W>
struct TokenWord {
  using P = PackFor<T, W == 1>;
  static constexpr int kPairs = (W + 1) / 2;    // pairs per slot
  static constexpr int kChans = W == 1 ? 2 : 1;  // channels per slot
  typename P::Word w[kPairs];
  // p: the slot's first channel; n: how many of its channels there are; step to the next one
  __device__ __forceinline__ void load(const T* p, int n, long long step) {
    if constexpr (W == 1) {
      const T a = n > 0 ? *p : from_acc<T>(0.f), b = n > 1 ? p[step] : from_acc<T>(0.f);
      if constexpr (sizeof(T) == 4) w[0] = make_float2(a, b);
      else w[0] = Halves{reinterpret_cast<const uint16_t&>(a), reinterpret_cast<const uint16_t&>(b)};
    } else if constexpr (sizeof(T) == 4) {
      w[0] = n > 0 ? *reinterpret_cast<const float2*>(p) : make_float2(0.f, 0.f);
    } else if constexpr (W == 4) {
      const uint2 q = n > 0 ? *reinterpret_cast<const uint2*>(p) : make_uint2(0u, 0u);
      w[0] = q.x;
      w[1] = q.y;
    } else {
      w[0] = n > 0 ? *reinterpret_cast<const uint32_t*>(p) : 0u;
    }
  }
  __device__ __forceinline__ void again() {
#pragma unroll
    for (int i = 0; i < kPairs; ++i) renew(w[i]);
  }
  static __device__ __forceinline__ void store(T* p, int n, long long step, const float2* f) {
    if constexpr (W == 1) {
      *p = from_acc<T>(f[0].x);
      if (n > 1) p[step] = from_acc<T>(f[0].y);
    } else if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float2*>(p) = f[0];
    } else if constexpr (W == 4) {
      *reinterpret_cast<uint2*>(p) = make_uint2(P::make(f[0]), P::make(f[1]));
    } else {
      *reinterpret_cast<uint32_t*>(p) = P::make(f[0]);
    }
  }
};

// Channels per thread: 32 registers of packed x.
template <typename T, int W>
constexpr int chan_cpt() {
  return W * (int)sizeof(T) == 8 ? 16 : 32;
}

// p + step as a value of its own: the products k * step of an unrolled loop would
// otherwise be kept over the loop about it, 64 registers.
template <typename T>
__device__ __forceinline__ void advance(T*& p, long long step) {
  p += step;
  asm volatile("" : "+l"(p));
}

// Shared-memory loads that stay where they are written: hoisted out of the loop over
// tiles, a thread's parameters would take its registers.
__device__ __forceinline__ float4 lds4(const float4* p) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(smem_u32(p)));
  return v;
}
__device__ __forceinline__ float2 lds2(const float2* p) {
  float2 v;
  asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(smem_u32(p)));
  return v;
}

// Joins S warps' (x, y) pairs per token through shared memory: join(token's S pairs)
// runs in one thread per token, spread over the warps, and every thread reads the results of
// its W tokens.  red: [S][W][32] pairs, then [W][32] results; the first barrier of the
// next use separates reading these results from writing those.
template <int W, typename J>
__device__ __forceinline__ void join_warps(float2 (&mine)[W], float2* red, int s, int S, int lane, J join) {
#pragma unroll
  for (int j = 0; j < W; ++j) red[(s * W + j) * 32 + lane] = mine[j];
  __syncthreads();
  float2* res = red + S * W * 32;
  for (int j = s; j < W; j += S) res[j * 32 + lane] = join(red + j * 32 + lane, W * 32);
  __syncthreads();
#pragma unroll
  for (int j = 0; j < W; ++j) mine[j] = res[j * 32 + lane];
}
// component j of pairs of tokens (W = 1: a sum over the pair of channels is one number)
template <int W>
__device__ __forceinline__ float token(const float2* p, int j) {
  return W == 1 ? p[0].x : (j & 1) ? p[j / 2].y : p[j / 2].x;
}
template <int W>
__device__ __forceinline__ void set_token(float2* p, int j, float v) {
  if (W == 1) p[0] = f2(v);
  else if (j & 1) p[j / 2].y = v;
  else p[j / 2].x = v;
}
// after sums over slots: W = 1 adds its two channels
template <int W>
__device__ __forceinline__ void fold_slot(float2* p) {
  if (W == 1) p[0] = f2(p[0].x + p[0].y);
}

// LOOP: more channels than S warps hold at once: a warp goes through its share CPT at a time,
// once for the statistics and once more (from L2) for y.
template <typename T, int W, int THREADS, bool LOOP>
__global__ void __launch_bounds__(THREADS, THREADS == 256 ? 3 : 1) ln_chan_fwd_kernel(LnArgs a) {
  using Word = TokenWord<T, W>;
  using P = typename Word::P;
  constexpr int CPT = chan_cpt<T, W>(), kPairs = Word::kPairs, kChans = Word::kChans, kSlots = CPT / kChans;
  extern __shared__ __align__(16) float ln_sm[];  // [C] (w, w, b, b) unless LOOP, then [P] x join_warps' pairs
  const int lane = threadIdx.x, s = threadIdx.y, S = blockDim.y, tiles_cta = blockDim.z;
  float4* par = reinterpret_cast<float4*>(ln_sm);
  if (!LOOP) {
    for (int c = threadIdx.x + 32 * (threadIdx.y + S * threadIdx.z); c < a.C; c += 32 * S * tiles_cta) {
      const float w = load_param(a.w, a.pdt, c, 1.f), b = load_param(a.b, a.pdt, c, 0.f);
      par[c] = make_float4(w, w, b, b);
    }
  }
  float2* red = reinterpret_cast<float2*>(par + (LOOP ? 0 : a.C)) + threadIdx.z * (S + 1) * W * 32;
  __syncthreads();
  const long long per = (a.inner + 32 * W - 1) / (32 * W), tiles = a.outer * per;
  const float rc = 1.f / (float)a.C;
  const int share = a.C / S, more = a.C - share * S;  // warp i has share channels, one more where i < more
  const int all = share + (s < more ? 1 : 0);
  // (w, w, b, b) of this warp's slot from channel k on; W = 1: of two channels
  const auto params = [&](int k, bool two) {
    const int c = k * S + s;
    float4 wb;
    if (LOOP) {
      wb = make_float4(load_param(a.w, a.pdt, c, 1.f), 0.f, load_param(a.b, a.pdt, c, 0.f), 0.f);
      wb.y = two ? load_param(a.w, a.pdt, c + S, 1.f) : wb.x;
      wb.w = two ? load_param(a.b, a.pdt, c + S, 0.f) : wb.z;
    } else {
      wb = lds4(par + c);
      if (two) {
        const float4 next = lds4(par + c + S);
        wb.y = next.y;
        wb.w = next.w;
      }
    }
    return wb;
  };
  for (long long base = (long long)blockIdx.x * tiles_cta; base < tiles; base += (long long)gridDim.x * tiles_cta) {
    const long long tile = base + threadIdx.z;
    const long long o = tile / per, v = (tile - o * per) * (32 * W) + lane * W;
    const bool in = tile < tiles && v < a.inner;  // inner is a multiple of W
    const long long at = (o * a.C + s) * a.inner + v, step = (long long)S * a.inner;
    Word x[kSlots];
    const auto load = [&](int first) {  // this warp's channels from `first` on
      const T* px = static_cast<const T*>(a.x) + at + first * step;
#pragma unroll
      for (int k = 0; k < kSlots; ++k, advance(px, step * kChans)) x[k].load(px, in ? all - first - k * kChans : 0, step);
    };
    // this warp's mean and squares about it; the pieces and the warps' join (Chan, Golub and LeVeque)
    float2 nm[kPairs], m2[kPairs];
#pragma unroll
    for (int j = 0; j < kPairs; ++j) nm[j] = m2[j] = make_float2(0.f, 0.f);
    for (int first = 0; first < (LOOP ? all : 1); first += CPT) {
      const int mine = LOOP ? min(CPT, all - first) : all;
      load(first);
      float2 pm[kPairs], p2[kPairs];
#pragma unroll
      for (int j = 0; j < kPairs; ++j) pm[j] = p2[j] = make_float2(0.f, 0.f);
#pragma unroll
      for (int k = 0; k < kSlots; ++k)
#pragma unroll
        for (int j = 0; j < kPairs; ++j) pm[j] = P::plus(x[k].w[j], pm[j]);
      fold_slot<W>(pm);
#pragma unroll
      for (int j = 0; j < kPairs; ++j) pm[j] = __fmul2_rn(pm[j], f2(-1.f / (float)mine));
#pragma unroll
      for (int k = 0; k < kSlots; ++k)
        if (k * kChans < mine) {
          x[k].again();
#pragma unroll
          for (int j = 0; j < kPairs; ++j) {
            float2 d = P::plus(x[k].w[j], pm[j]);
            if (W == 1 && k * kChans + 1 >= mine) d.y = 0.f;
            p2[j] = __ffma2_rn(d, d, p2[j]);
          }
        }
      fold_slot<W>(p2);
      const float na = (float)first, nb = (float)mine, share_b = nb / (na + nb);
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        if (!LOOP) {
          nm[j] = pm[j];
          m2[j] = p2[j];
        } else {
          const float2 d = __fadd2_rn(pm[j], make_float2(-nm[j].x, -nm[j].y));
          nm[j] = __ffma2_rn(d, f2(share_b), nm[j]);
          m2[j] = __fadd2_rn(m2[j], __ffma2_rn(__fmul2_rn(d, d), f2(na * share_b), p2[j]));
        }
      }
    }
    float2 rstd[kPairs];
    float2 st[W];
#pragma unroll
    for (int j = 0; j < W; ++j) st[j] = make_float2(token<W>(nm, j), token<W>(m2, j));
    if (S > 1) {
      join_warps<W>(st, red, s, S, lane, [=](const float2* p, int stride) {
        float sum = 0.f, sq = 0.f;
        for (int i = 0; i < S; ++i) sum = fmaf((float)(share + (i < more ? 1 : 0)), p[i * stride].x, sum);
        const float m = sum * rc;  // of -x, as nm
        for (int i = 0; i < S; ++i) {
          const float d = p[i * stride].x - m;
          sq += fmaf((float)(share + (i < more ? 1 : 0)) * d, d, p[i * stride].y);
        }
        return make_float2(m, sq);
      });
    }
#pragma unroll
    for (int j = 0; j < W; ++j) {
      st[j].y = rsqrtf(st[j].y * rc + a.eps);
      set_token<W>(nm, j, st[j].x);
      set_token<W>(rstd, j, st[j].y);
    }
    if (in) {
      for (int first = 0; first < (LOOP ? all : 1); first += CPT) {
        const int mine = LOOP ? min(CPT, all - first) : all;
        if (LOOP) load(first);
        T* y = static_cast<T*>(a.y) + at + first * step;
#pragma unroll
        for (int k = 0; k < kSlots; ++k, advance(y, step * kChans))
          if (k * kChans < mine) {
            const float4 wb = params(first + k * kChans, W == 1 && k * kChans + 1 < mine);
            float2 f[kPairs];
            x[k].again();
#pragma unroll
            for (int j = 0; j < kPairs; ++j)
              f[j] = __ffma2_rn(__fmul2_rn(P::plus(x[k].w[j], nm[j]), rstd[j]), make_float2(wb.x, wb.y),
                                make_float2(wb.z, wb.w));
            Word::store(y, mine - k * kChans, step, f);
          }
      }
      if (a.stats != nullptr && s == 0) {
#pragma unroll
        for (int j = 0; j < W; ++j) a.stats[o * a.inner + v + j] = make_float2(-st[j].x, st[j].y);
      }
    }
  }
}

// Sums over the 32 lanes of N values each: lane l returns the sum of value l % N.  Halves
// change places at distances N / 2 .. 1: N - 1 shuffles (and one for N = 16) instead of 5 N.
template <int N>
__device__ __forceinline__ float transpose_sum(float (&v)[N], int lane) {
#pragma unroll
  for (int o = N / 2; o > 0; o >>= 1) {
    const bool up = lane & o;
#pragma unroll
    for (int i = 0; i < o; ++i) {
      const float send = up ? v[i] : v[i + o], keep = up ? v[i + o] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
    }
  }
  if (N == 16) v[0] += __shfl_xor_sync(0xffffffffu, v[0], 16);
  return v[0];
}

// LOOP: as forward; x and dy are read twice, and a channel's weight-grad sums are kept in
// shared memory by the lane that owns it.
template <typename T, int W, int THREADS, bool LOOP>
__global__ void __launch_bounds__(THREADS, THREADS == 256 ? 2 : 1) ln_chan_bwd_kernel(LnArgs a) {
  using Word = TokenWord<T, W>;
  using P = typename Word::P;
  constexpr int CPT = chan_cpt<T, W>(), kPairs = Word::kPairs, kChans = Word::kChans, kSlots = CPT / kChans;
  // [C] (w, w), or (dw, db) where LOOP; then [P] x join_warps' pairs
  extern __shared__ __align__(16) float ln_sm[];
  grid_dependents_go();
  const int lane = threadIdx.x, s = threadIdx.y, S = blockDim.y, tiles_cta = blockDim.z;
  float2* par = reinterpret_cast<float2*>(ln_sm);
  for (int c = threadIdx.x + 32 * (threadIdx.y + S * threadIdx.z); c < a.C; c += 32 * S * tiles_cta)
    par[c] = LOOP ? make_float2(0.f, 0.f) : f2(load_param(a.w, a.pdt, c, 1.f));
  float2* red = par + a.C + threadIdx.z * (S + 1) * W * 32;
  __syncthreads();
  const long long per = (a.inner + 32 * W - 1) / (32 * W), tiles = a.outer * per;
  const float rc = 1.f / (float)a.C;
  const int all = a.C / S + (s < a.C % S ? 1 : 0);
  const auto weight = [&](int k, bool two) {  // of this warp's slot from channel k on
    const int c = k * S + s;
    if (LOOP) return make_float2(load_param(a.w, a.pdt, c, 1.f), load_param(a.w, a.pdt, two ? c + S : c, 1.f));
    float2 w = lds2(par + c);
    if (two) w.y = lds2(par + c + S).y;
    return w;
  };
  float dw = 0.f, db = 0.f;  // of channel (lane % CPT) * S + s
  for (long long base = (long long)blockIdx.x * tiles_cta; base < tiles; base += (long long)gridDim.x * tiles_cta) {
    const long long tile = base + threadIdx.z;
    const long long o = tile / per, v = (tile - o * per) * (32 * W) + lane * W;
    const bool in = tile < tiles && v < a.inner;
    const long long at = (o * a.C + s) * a.inner + v, step = (long long)S * a.inner;
    Word x[kSlots], d[kSlots];
    const auto load = [&](int first) {
      const T *px = static_cast<const T*>(a.x) + at + first * step, *pd = static_cast<const T*>(a.dy) + at + first * step;
#pragma unroll
      for (int k = 0; k < kSlots; ++k, advance(px, step * kChans), advance(pd, step * kChans)) {
        x[k].load(px, in ? all - first - k * kChans : 0, step);
        d[k].load(pd, in ? all - first - k * kChans : 0, step);
      }
    };
    if (!LOOP) load(0);
    float2 nm[kPairs], r[kPairs], s1[kPairs], s2[kPairs];
#pragma unroll
    for (int j = 0; j < W; ++j) {
      const float2 st = in ? a.stats[o * a.inner + v + j] : make_float2(0.f, 0.f);
      set_token<W>(nm, j, -st.x);
      set_token<W>(r, j, st.y);
    }
#pragma unroll
    for (int j = 0; j < kPairs; ++j) s1[j] = s2[j] = make_float2(0.f, 0.f);
    for (int first = 0; first < (LOOP ? all : 1); first += CPT) {
      const int mine = LOOP ? min(CPT, all - first) : all;
      if (LOOP) load(first);
#pragma unroll
      for (int k = 0; k < kSlots; ++k)
        if (k * kChans < mine) {
          const float2 w = weight(first + k * kChans, W == 1 && k * kChans + 1 < mine);
#pragma unroll
          for (int j = 0; j < kPairs; ++j) {
            // sum of g (x - mean): the common r is multiplied once, below.  An absent second
            // channel (W = 1) has dy = 0.
            const float2 gw = __fmul2_rn(P::value(d[k].w[j]), w);
            s1[j] = __fadd2_rn(s1[j], gw);
            s2[j] = __ffma2_rn(gw, P::plus(x[k].w[j], nm[j]), s2[j]);
          }
        }
    }
    fold_slot<W>(s1);
    fold_slot<W>(s2);
    if (S > 1) {
      float2 sums[W];
#pragma unroll
      for (int j = 0; j < W; ++j) sums[j] = make_float2(token<W>(s1, j), token<W>(s2, j));
      join_warps<W>(sums, red, s, S, lane, [=](const float2* p, int stride) {
        float2 t = p[0];
        for (int i = 1; i < S; ++i) t = __fadd2_rn(t, p[i * stride]);
        return t;
      });
#pragma unroll
      for (int j = 0; j < W; ++j) {
        set_token<W>(s1, j, sums[j].x);
        set_token<W>(s2, j, sums[j].y);
      }
    }
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {
      s1[j] = __fmul2_rn(s1[j], f2(-rc));                    // -mean(g)
      s2[j] = __fmul2_rn(__fmul2_rn(s2[j], r[j]), f2(-rc));  // -mean(g xh)
    }
    for (int first = 0; first < (LOOP ? all : 1); first += CPT) {
      const int mine = LOOP ? min(CPT, all - first) : all;
      if (LOOP) load(first);
      float pw[CPT], pb[CPT];
      T* dx = static_cast<T*>(a.y) + at + first * step;
#pragma unroll
      for (int k = 0; k < kSlots; ++k, advance(dx, step * kChans)) {
        float2 tw = make_float2(0.f, 0.f), tb = tw;
        if (k * kChans < mine) {
          const float2 w = weight(first + k * kChans, W == 1 && k * kChans + 1 < mine);
          float2 f[kPairs];
          x[k].again();
          d[k].again();
#pragma unroll
          for (int j = 0; j < kPairs; ++j) {
            const float2 g = P::value(d[k].w[j]), xh = __fmul2_rn(P::plus(x[k].w[j], nm[j]), r[j]);
            tw = __ffma2_rn(g, xh, tw);
            tb = __fadd2_rn(tb, g);
            f[j] = __fmul2_rn(__ffma2_rn(xh, s2[j], __ffma2_rn(g, w, s1[j])), r[j]);
          }
          if (in) Word::store(dx, mine - k * kChans, step, f);
        }
        if constexpr (W == 1) {
          pw[2 * k] = tw.x;
          pw[2 * k + 1] = tw.y;
          pb[2 * k] = tb.x;
          pb[2 * k + 1] = tb.y;
        } else {
          pw[k] = tw.x + tw.y;
          pb[k] = tb.x + tb.y;
        }
      }
      if (a.part != nullptr) {
        const float2 t = make_float2(transpose_sum<CPT>(pw, lane), transpose_sum<CPT>(pb, lane));
        if (!LOOP) {
          dw += t.x;
          db += t.y;
        } else if (lane < mine) {  // LOOP has one tile per CTA at a time: this warp's alone
          float2* acc = par + (first + lane) * S + s;
          *acc = __fadd2_rn(*acc, t);
        }
      }
    }
  }
  if (a.part == nullptr) return;
  // the CTA's tiles, in order, then one partial per CTA
  __syncthreads();
  float* part = a.part + (long long)blockIdx.x * 2 * a.C;
  if (LOOP) {
    for (int c = threadIdx.x + 32 * threadIdx.y; c < a.C; c += 32 * S) {
      part[c] = par[c].x;
      part[a.C + c] = par[c].y;
    }
    return;
  }
  float2* acc = par + a.C;  // [P][S][32]
  acc[(threadIdx.z * S + s) * 32 + lane] = make_float2(dw, db);
  __syncthreads();
  if (threadIdx.z == 0 && lane < all) {
    float2 t = acc[s * 32 + lane];
    for (int p = 1; p < tiles_cta; ++p) t = __fadd2_rn(t, acc[(p * S + s) * 32 + lane]);
    part[lane * S + s] = t.x;
    part[a.C + lane * S + s] = t.y;
  }
}

// ------------------------------ host side ------------------------------
// How a call runs.  kAny: rows that do not fit into registers.
enum LnForm { kRows, kChan, kAny };
struct LnPlan {
  LnForm form;
  int vec;          // kRows: elements per word; kChan: tokens per word
  int ept;          // kRows: elements per thread
  int G;            // kRows: threads per row
  int threads;      // kRows: of a CTA
  int S, P;         // kChan: warps per tile, tiles per CTA
  bool loop;        // kChan: more channels than the warps hold
  long long units;  // CTA-sized pieces of work
};

// Rows: a power of two of threads with 8 elements each up to 256 columns, whole warps with 16
// up to 4096, then with 32 as many as the CTA has: 8192 columns.  (16 against 32 per thread:
// 4096 x 4096 fp32 forward 25 us against 36, backward 44 against 69; 16384 x 1024 bf16
// forward 17.8 against 16.8, backward 28 against 35.)
LnPlan plan_rows(long long tokens, int C, int vec) {
  LnPlan p{};
  p.form = kAny;
  // single elements take a register and a predicate each: 8 per thread, on more threads
  if (C > kRowThreads * (vec == 1 ? 8 : 32)) return p;
  p.form = kRows;
  p.vec = vec;
  p.ept = vec == 1 || C <= 256 ? 8 : C <= kRowThreads * 16 ? 16 : 32;
  const int need = (C + p.ept - 1) / p.ept;
  p.G = 1;
  while (p.G < need && p.G < 32) p.G *= 2;
  if (need > 32) p.G = (need + 31) / 32 * 32;
  p.threads = kRowThreads / p.G * p.G;
  const int rows = p.threads / p.G;
  p.units = (tokens + rows - 1) / rows;
  return p;
}

// Channels first: the widest word that the alignment allows and whose tile has enough
// warps for C: 32 forward, 16 backward (its threads hold x and dy); more channels than any
// holds are gone through in a loop, with the widest word.  Backward, LOOP keeps 8 bytes per
// channel in shared memory: up to 16384 of them.
LnPlan plan_chan(long long outer, long long inner, int C, size_t esz, size_t align, bool bwd) {
  LnPlan p{};
  const int most = bwd ? 16 : 32;
  p.form = kChan;
  int widest = 1;
  for (int w = (int)(8 / esz); w >= 1; w /= 2) {
    if (inner % w != 0 || align % (w * esz) != 0) continue;
    widest = std::max(widest, w);
    const int cpt = w * (int)esz == 8 ? 16 : 32;
    p.S = (C + cpt - 1) / cpt;
    if (p.S > most) continue;
    p.vec = w;
    p.P = std::max(1, 4 / p.S);
    p.units = (outer * ((inner + 32 * w - 1) / (32 * w)) + p.P - 1) / p.P;
    return p;
  }
  p.loop = true;
  p.vec = widest;
  p.S = most;
  p.P = 1;
  p.units = outer * ((inner + 32 * widest - 1) / (32 * widest));
  return p;
}

template <typename T>
LnPlan plan_ln(const LnArgs& a, bool bwd) {
  // the largest power of two that divides every address, up to 16
  const uintptr_t bits = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.y) |
                         reinterpret_cast<uintptr_t>(a.dy) | 16;
  const size_t align = (size_t)(bits & (~bits + 1));
  if (a.inner > 1) return plan_chan(a.outer, a.inner, a.C, sizeof(T), align, bwd);
  constexpr int V = 16 / sizeof(T);
  int vec = 1;
  if (a.C % V == 0 && align == 16) vec = V;
  else if (sizeof(T) == 2 && a.C % 2 == 0 && align >= 4) vec = 2;
  return plan_rows(a.tokens, a.C, vec);
}

// Most weight-grad partials that a call makes: one per CTA of the backward kernel, four
// CTAs per SM; at least four tokens each, so that the partials stay small beside the data, and
// 64 MB of them or one per SM.  Rows past the register kernels: enough CTAs for the GPU over
// the columns and the parts.
int dw_parts(long long tokens, int C, long long inner) {
  long long most = std::min(kSms * 4LL, std::max<long long>(kSms, (1LL << 23) / C));
  if (inner == 1 && C > kRowThreads * 32) most = std::max(1LL, kSms * 8LL / ((C + 31) / 32));
  return (int)std::max(1LL, std::min(most, (tokens + 3) / 4));
}

// Launches the rows kernels for a plan's vec and ept.
template <typename T, int VEC, int EPT, int R>
int launch_rows(const LnArgs& a, const LnPlan& p, bool bwd, int parts, cudaStream_t s) {
  const size_t param = RowParam<T, VEC, EPT>::smem_bytes(p.G);
  if (!bwd) {
    auto kern = ln_rows_fwd_kernel<T, VEC, EPT, R>;
    const size_t smem = kBlockRows<T, VEC, R> ? 3 * (size_t)block_bytes<T>(p.threads / p.G * R, a.C) : 2 * param;
    const int st = ensure_smem(kern, smem);
    if (st != MEDNEXT_OK) return st;
    const long long cap = kSms * 2LL;  // resident by the launch bounds
    kern<<<(unsigned)std::min((p.units + R - 1) / R, cap), p.threads, smem, s>>>(a, p.G);
  } else {
    constexpr int RB = R > 2 ? 2 : 1;
    auto kern = ln_rows_bwd_kernel<T, VEC, EPT, RB>;
    const int slots = p.G < 32 ? p.threads / 32 : p.threads / p.G;
    const size_t held = kBlockRows<T, VEC, RB> ? 5 * (size_t)block_bytes<T>(p.threads / p.G * RB, a.C) : param;
    const size_t smem = std::max(held, a.part != nullptr ? (size_t)slots * 2 * a.C * sizeof(float) : 0);
    const int st = ensure_smem(kern, smem);
    if (st != MEDNEXT_OK) return st;
    kern<<<parts, p.threads, smem, s>>>(a, p.G);
  }
  return record_launch();
}
template <typename T, int VEC>
int launch_rows_vec(const LnArgs& a, const LnPlan& p, bool bwd, int parts, cudaStream_t s) {
  // rows in flight per thread (half as many backward), once every SM has that much to do
  const bool many = p.units >= kSms * 12;
  if (VEC == 1 || p.ept == 8)
    return many ? launch_rows<T, VEC, 8, 4>(a, p, bwd, parts, s) : launch_rows<T, VEC, 8, 1>(a, p, bwd, parts, s);
  if constexpr (VEC > 1) {
    if (p.ept == 16)
      return many ? launch_rows<T, VEC, 16, 2>(a, p, bwd, parts, s) : launch_rows<T, VEC, 16, 1>(a, p, bwd, parts, s);
    return launch_rows<T, VEC, 32, 1>(a, p, bwd, parts, s);
  }
  return MEDNEXT_ERR_UNSUPPORTED;  // not reached
}
template <typename T>
int launch_rows_any_vec(const LnArgs& a, const LnPlan& p, bool bwd, int parts, cudaStream_t s) {
  if (p.vec == 1) return launch_rows_vec<T, 1>(a, p, bwd, parts, s);
  if constexpr (sizeof(T) == 2)
    if (p.vec == 2) return launch_rows_vec<T, 2>(a, p, bwd, parts, s);
  return launch_rows_vec<T, 16 / sizeof(T)>(a, p, bwd, parts, s);
}

template <typename T, int W, int FWD_THREADS, int BWD_THREADS, bool LOOP>
int launch_chan(const LnArgs& a, const LnPlan& p, bool bwd, int parts, cudaStream_t s) {
  const size_t red = (size_t)p.P * (p.S + 1) * W * 32 * sizeof(float2);
  const dim3 block(32, p.S, p.P);
  if (!bwd) {
    auto kern = ln_chan_fwd_kernel<T, W, FWD_THREADS, LOOP>;
    const size_t smem = (LOOP ? 0 : (size_t)a.C * sizeof(float4)) + red;
    const int st = ensure_smem(kern, smem);
    if (st != MEDNEXT_OK) return st;
    const long long cap = kSms * (long long)std::max(1, 24 / (p.S * p.P));  // resident: 24 warps
    kern<<<(unsigned)std::min(p.units, cap), block, smem, s>>>(a);
  } else {
    auto kern = ln_chan_bwd_kernel<T, W, BWD_THREADS, LOOP>;
    const size_t smem = (size_t)a.C * sizeof(float2) + red;
    const int st = ensure_smem(kern, smem);
    if (st != MEDNEXT_OK) return st;
    kern<<<parts, block, smem, s>>>(a);
  }
  return record_launch();
}
template <typename T, int W>
int launch_chan_word(const LnArgs& a, const LnPlan& p, bool bwd, int parts, cudaStream_t s) {
  if (p.loop) return launch_chan<T, W, 1024, 512, true>(a, p, bwd, parts, s);
  return p.S <= 8 ? launch_chan<T, W, 256, 256, false>(a, p, bwd, parts, s)
                  : launch_chan<T, W, 1024, 512, false>(a, p, bwd, parts, s);
}
template <typename T>
int launch_chan_any_word(const LnArgs& a, const LnPlan& p, bool bwd, int parts, cudaStream_t s) {
  if (p.vec == 1) return launch_chan_word<T, 1>(a, p, bwd, parts, s);
  if constexpr (sizeof(T) == 2)
    if (p.vec == 4) return launch_chan_word<T, 4>(a, p, bwd, parts, s);
  return launch_chan_word<T, 2>(a, p, bwd, parts, s);
}

template <typename T>
int ln_fwd(const LnArgs& a, cudaStream_t s) {
  const LnPlan p = plan_ln<T>(a, false);
  if (p.form == kRows) return launch_rows_any_vec<T>(a, p, false, 0, s);
  if (p.form == kChan) return launch_chan_any_word<T>(a, p, false, 0, s);
  ln_rows_any_fwd_kernel<T><<<(unsigned)std::min<long long>(a.tokens, kSms * 32), 256, 0, s>>>(a);
  return record_launch();
}

template <typename T>
int ln_bwd(const LnArgs& a, void* dw, void* db, cudaStream_t s) {
  const LnPlan p = plan_ln<T>(a, true);
  // one CTA per resident slot (the launch bounds leave 512 threads), one partial per CTA
  const int warps = p.form == kRows ? p.threads / 32 : std::max(1, p.S * p.P);
  const long long slots = (long long)kSms * std::max(1, 16 / warps);
  int st, parts = (int)std::min<long long>(std::min<long long>(dw_parts(a.tokens, a.C, a.inner), slots), std::max(1LL, p.units));
  if (p.form == kRows) {
    st = launch_rows_any_vec<T>(a, p, true, parts, s);
  } else if (p.form == kChan) {
    st = launch_chan_any_word<T>(a, p, true, parts, s);
  } else {
    const long long cols = (a.C + 31) / 32;
    parts = (int)std::min<long long>(dw_parts(a.tokens, a.C, 1), std::max(1LL, kSms * 8LL / cols));
    ln_rows_any_dx_kernel<T><<<(unsigned)std::min<long long>(a.tokens, kSms * 32), 256, 0, s>>>(a);
    st = record_launch();
    if (st != MEDNEXT_OK || a.part == nullptr) return st;
    ln_rows_any_dw_kernel<T><<<dim3((unsigned)cols, parts), 256, 0, s>>>(a, parts);
    st = record_launch();
  }
  if (st != MEDNEXT_OK || a.part == nullptr) return st;
  return launch_dependent(ln_fold_kernel, dim3((a.C + 31) / 32), dim3(1024), 0, s, (const float*)a.part, parts, a.C, dw,
                          db, a.pdt);
}

// Everything that both directions check.  Token and channel counts below 2^31 keep the
// kernels' channel indexes in 32 bits; element offsets are 64-bit.
int ln_check(int64_t outer, int64_t c, int64_t inner, int dtype, int param_dtype) {
  if (dtype != MEDNEXT_FLOAT32 && dtype != MEDNEXT_BFLOAT16 && dtype != MEDNEXT_FLOAT16) return MEDNEXT_ERR_BAD_DTYPE;
  if (param_dtype != MEDNEXT_FLOAT32 && param_dtype != dtype) return MEDNEXT_ERR_BAD_DTYPE;
  if (outer < 0 || inner < 0 || c <= 0 || c > ((int64_t)1 << 24)) return MEDNEXT_ERR_BAD_SHAPE;
  if (inner > 1 && c > kChanMost) return MEDNEXT_ERR_BAD_SHAPE;
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
