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
#include <type_traits>

#include "plan.h"
#include "pointwise_tma.cuh"
#include "tma_host.h"

namespace mednext {
namespace {

constexpr float kTinyMax = 127.f * 1.17549435e-38f;
constexpr int kI8MaxK = 131072;
constexpr int kI8MaxN = 1 << 22;
constexpr int kI8Sms = 148;

// The largest magnitude of a token as ordered bits: the bits of |x| as an unsigned
// number order as |x| does, infinity above every number and NaN above infinity.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

struct TokenScale {
  float scale;    // s_t
  float inverse;  // 127 / m_t, 0 where m_t is not finite
};
__device__ __forceinline__ float token_inverse(uint32_t max_bits) {
  return max_bits >= 0x7f800000u ? 0.f : __fdiv_rn(127.f, fmaxf(__uint_as_float(max_bits), kTinyMax));
}
__device__ __forceinline__ TokenScale token_scale(uint32_t max_bits) {
  const float m = max_bits >= 0x7f800000u ? __uint_as_float(max_bits) : fmaxf(__uint_as_float(max_bits), kTinyMax);
  return {__fdiv_rn(m, 127.f), token_inverse(max_bits)};
}
// ------------------------------ quantisation ------------------------------
// rint(v * inverse) as the low byte of the sum with 1.5 * 2^23 (the sum's unit is 1, so its
// rounding is the rint): two fp32 instructions in place of a conversion.  The product is
// rounded before the sum, as the definition says.  Scalar intrinsics: the packed
// fp32 x 2 product and sum were fused into one multiply-add, which rounds some of 10^4
// values the other way.
constexpr float kRint = 12582912.f;
__device__ __forceinline__ float2 scaled2(float2 v, float inverse_x, float inverse_y) {
  return make_float2(__fadd_rn(__fmul_rn(v.x, inverse_x), kRint), __fadd_rn(__fmul_rn(v.y, inverse_y), kRint));
}
// Four bytes of a token at once; a token without a scale (infinity or NaN in it) is masked
// to zeros by the caller.
__device__ __forceinline__ uint32_t low_bytes(float a, float b, float c, float d) {
  const uint32_t ab = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x0040);
  const uint32_t cd = __byte_perm(__float_as_uint(c), __float_as_uint(d), 0x0040);
  return __byte_perm(ab, cd, 0x5410);
}

// Packed pairs: the running maximum of magnitudes and the values.
template <typename T>
struct Mag {  // 16-bit types: two per word, their bits ordered as the numbers are
  using Word = uint32_t;
  using Max = uint32_t;
  static __device__ __forceinline__ Max join(Max m, Word w) { return __vmaxu2(m, w & 0x7fff7fffu); }
  static __device__ __forceinline__ uint32_t lo(Max m) { return abs_bits(unpack2<T>(m).x); }
  static __device__ __forceinline__ uint32_t hi(Max m) { return abs_bits(unpack2<T>(m).y); }
  static __device__ __forceinline__ float2 value(Word w) { return unpack2<T>(w); }
};
template <>
struct Mag<float> {
  using Word = float2;
  using Max = uint2;
  static __device__ __forceinline__ Max join(Max m, Word w) {
    return make_uint2(max(m.x, abs_bits(w.x)), max(m.y, abs_bits(w.y)));
  }
  static __device__ __forceinline__ uint32_t lo(Max m) { return m.x; }
  static __device__ __forceinline__ uint32_t hi(Max m) { return m.y; }
  static __device__ __forceinline__ float2 value(Word w) { return w; }
};

// Rows whose start and length are multiples of 16 bytes: G threads (a power of two up to 32)
// hold a row's NV 16-byte vectors each; x is read once.
template <typename T, int NV>
__global__ void __launch_bounds__(256) i8_quantize_rows_kernel(const T* __restrict__ x, int8_t* __restrict__ q,
                                                               float* __restrict__ scale, long long tokens, int K,
                                                               int pitch, int G) {
  using M = Mag<T>;
  constexpr int E = 16 / sizeof(T), kPairs = E / 2;
  grid_dependents_go();
  const int groups = 256 / G, gi = threadIdx.x / G, gl = threadIdx.x - gi * G;
  // uniform over the CTA: every lane takes part in the shuffles
  for (long long t0 = (long long)blockIdx.x * groups; t0 < tokens; t0 += (long long)gridDim.x * groups) {
    const long long t = t0 + gi;
    typename M::Word w[NV][kPairs];
    typename M::Max m{};
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * G + gl) * E;
      const uint4 r = t < tokens && c < K ? *reinterpret_cast<const uint4*>(x + t * K + c) : make_uint4(0, 0, 0, 0);
      memcpy(w[v], &r, 16);
    }
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int i = 0; i < kPairs; ++i) m = M::join(m, w[v][i]);
    uint32_t most = max(M::lo(m), M::hi(m));
    for (int o = G >> 1; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
    if (t >= tokens) continue;
    const TokenScale s = token_scale(most);
    const uint32_t keep = most >= 0x7f800000u ? 0u : 0xffffffffu;
    if (gl == 0) scale[t] = s.scale;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * G + gl) * E;
      if (c >= pitch) continue;  // columns K .. pitch get the zeros that were not loaded
      uint32_t b[E / 4];
#pragma unroll
      for (int i = 0; i < E / 4; ++i) {
        const float2 f = scaled2(M::value(w[v][2 * i]), s.inverse, s.inverse),
                     g = scaled2(M::value(w[v][2 * i + 1]), s.inverse, s.inverse);
        b[i] = low_bytes(f.x, f.y, g.x, g.y) & keep;
      }
      if constexpr (E == 8) *reinterpret_cast<uint2*>(q + t * pitch + c) = make_uint2(b[0], b[1]);
      else *reinterpret_cast<uint32_t*>(q + t * pitch + c) = b[0];
    }
  }
}

// 16 channels of W tokens (packed pairs of tokens for W = 2) to 16 bytes per token.
template <typename T, int W>
__device__ __forceinline__ void quantize16(const uint32_t* w, const TokenScale (&ts)[W], uint32_t (&b)[W][4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 f[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t word = w[i * 4 + e];
      if constexpr (W == 2) f[e] = unpack2<T>(word);
      else if constexpr (sizeof(T) == 4) f[e] = make_float2(__uint_as_float(word), 0.f);
      else f[e] = make_float2(unpack2<T>(word).x, 0.f);
      f[e] = scaled2(f[e], ts[0].inverse, ts[W - 1].inverse);
    }
    b[0][i] = low_bytes(f[0].x, f[1].x, f[2].x, f[3].x);
    if constexpr (W == 2) b[1][i] = low_bytes(f[0].y, f[1].y, f[2].y, f[3].y);
  }
}

// Channels first: a lane owns W neighbouring tokens (two 16-bit elements of a word, else one)
// and CH channels in a row of them.  TX lanes lie along the tokens, 32 / TX along further
// channels, so that a warp has a piece of 32 / TX * CH channels; warp s of a tile's S takes
// the pieces s, s + S, ..  Each load is a segment of a channel's row, each token's bytes are
// 16-byte stores: the transpose to token rows costs no shared memory.  With one piece per
// warp x is read once; else the pieces are read again (from L2) to be scaled.
// blockDim = (32, S, P), P tiles side by side.
//
// TX = 32, CH = 32 is for many tokens.  Few tokens (deep levels) leave most SMs without a tile
// of that size: TX = 8, CH = 16 makes four times as many, in 16- or 32-byte segments
// (2048 channels x 512 voxels bf16: 14.9 -> 6.3 us).
template <typename T, int W, int TX, int CH>
__global__ void __launch_bounds__(1024) i8_quantize_chan_kernel(const T* __restrict__ x, int8_t* __restrict__ q,
                                                                float* __restrict__ scale, int outer, int inner,
                                                                int K, int pitch) {
  constexpr int kPiece = 32 / TX * CH;
  extern __shared__ uint32_t i8_max[];  // [2][P][S][W][TX]
  grid_dependents_go();
  const int lane = threadIdx.x, s = threadIdx.y, S = blockDim.y, P = blockDim.z;
  const int tx = lane % TX, cy = lane / TX;
  const int per = (inner + TX * W - 1) / (TX * W), pieces = (pitch + kPiece - 1) / kPiece;  // pitch >= K
  const long long tiles = (long long)outer * per;
  int turn = 0;
  for (long long base = (long long)blockIdx.x * P; base < tiles; base += (long long)gridDim.x * P) {
    const long long tile = base + threadIdx.z;
    const int o = (int)(tile / per), v = (int)(tile - (long long)o * per) * (TX * W) + tx * W;
    const bool in = tile < tiles && v < inner;  // inner is even where W = 2
    const T* px = x + (long long)o * K * inner + v;
    uint32_t w[CH];
    const auto load = [&](int piece) {
#pragma unroll
      for (int k = 0; k < CH; ++k) {
        const int c = piece * kPiece + cy * CH + k;
        const bool ok = in && c < K;
        const T* p = px + (long long)c * inner;
        if constexpr (W == 2) w[k] = ok ? *reinterpret_cast<const uint32_t*>(p) : 0u;
        else if constexpr (sizeof(T) == 4) w[k] = ok ? __float_as_uint(*p) : 0u;
        else w[k] = ok ? (uint32_t)*reinterpret_cast<const uint16_t*>(p) : 0u;
      }
    };
    uint32_t m = 0;  // magnitudes: W = 2 two 16-bit ones, else one
    for (int piece = s; piece < pieces; piece += S) {
      load(piece);
#pragma unroll
      for (int k = 0; k < CH; ++k) {
        if constexpr (W == 2) m = __vmaxu2(m, w[k] & 0x7fff7fffu);
        else m = max(m, w[k] & (sizeof(T) == 4 ? 0x7fffffffu : 0x7fffu));
      }
    }
#pragma unroll
    for (int d = TX; d < 32; d *= 2) {
      const uint32_t other = __shfl_xor_sync(0xffffffffu, m, d);
      m = W == 2 ? __vmaxu2(m, other) : max(m, other);
    }
    uint32_t most[W];
    if constexpr (W == 2) {
      most[0] = Mag<T>::lo(m);
      most[W - 1] = Mag<T>::hi(m);
    } else if constexpr (sizeof(T) == 4) {
      most[0] = m;
    } else {
      most[0] = abs_bits(unpack2<T>(m).x);
    }
    if (S > 1) {
      uint32_t* r = i8_max + (turn * P + threadIdx.z) * S * W * TX;
      turn ^= 1;
      if (cy == 0) {
#pragma unroll
        for (int j = 0; j < W; ++j) r[(s * W + j) * TX + tx] = most[j];
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < W; ++j)
        for (int i = 0; i < S; ++i) most[j] = max(most[j], r[(i * W + j) * TX + tx]);
    }
    TokenScale ts[W];
#pragma unroll
    for (int j = 0; j < W; ++j) ts[j] = token_scale(most[j]);
    if (in) {
      const long long t = (long long)o * inner + v;
      if (s == 0 && cy == 0) {
#pragma unroll
        for (int j = 0; j < W; ++j) scale[t + j] = ts[j].scale;
      }
      for (int piece = s; piece < pieces; piece += S) {
        if (pieces > S) load(piece);
#pragma unroll
        for (int h = 0; h < CH / 16; ++h) {
          const int c = piece * kPiece + cy * CH + h * 16;
          if (c >= pitch) break;
          uint32_t b[W][4];
          quantize16<T, W>(w + h * 16, ts, b);
#pragma unroll
          for (int j = 0; j < W; ++j) {
            const uint32_t keep = most[j] >= 0x7f800000u ? 0u : 0xffffffffu;
            *reinterpret_cast<uint4*>(q + (t + j) * pitch + c) =
                make_uint4(b[j][0] & keep, b[j][1] & keep, b[j][2] & keep, b[j][3] & keep);
          }
        }
      }
    }
    __syncwarp();  // whole again for the next tile's shuffles
  }
}

// Rows of any alignment and width: one token per warp at a time, four neighbouring values per
// lane and step, so that their bytes are one store.  128 kSteps values stay in registers;
// longer rows are read again (from L1 / L2) to be scaled.
// BLOCK: eight rows of 16-bit data at a time through shared memory, the next eight under way
// (100000 x 777 fp16: 66 us, from global memory 77; 30000 x 2001 bf16 53, 75; 10000 x 97 4.3, 3.6).
template <typename T, bool BLOCK, int kSteps>
__global__ void __launch_bounds__(256) i8_quantize_any_kernel(const T* __restrict__ x, int8_t* __restrict__ q,
                                                              float* __restrict__ scale, long long tokens, int K,
                                                              int pitch) {
  extern __shared__ __align__(16) uint8_t i8_rows[];  // BLOCK: [2] blocks
  grid_dependents_go();
  const int lane = threadIdx.x & 31, bytes = block_bytes<T>(8, K);
  int buf = 0;
  const auto fetch = [&](long long t0) {
    if (t0 < tokens) RowBlock<T>::fetch(i8_rows + buf * bytes, x + t0 * K, (int)min(8LL, tokens - t0) * K);
  };
  if (BLOCK) fetch((long long)blockIdx.x * 8);
  // the CTA's warps go their own ways, or together from block to block
  const int warp = threadIdx.x >> 5;
  for (long long t = (long long)blockIdx.x * 8 + warp; (BLOCK ? t - warp : t) < tokens; t += (long long)gridDim.x * 8) {
    const T* p = x + t * K;
    if constexpr (BLOCK) {
      const long long t0 = t - warp;
      RowBlock<T>::arrived();
      __syncthreads();  // this block is there, the last one has been read
      p = RowBlock<T>::first(i8_rows + buf * bytes, x + t0 * K) + warp * K;
      buf ^= 1;
      fetch(t0 + (long long)gridDim.x * 8);
      if (t >= tokens) continue;
    }
    const auto value = [&](int k) { return k < K ? to_acc<T>(p[k]) : 0.f; };
    float v[kSteps][4];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < kSteps; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[i][e] = value((i * 32 + lane) * 4 + e);
        m = max(m, abs_bits(v[i][e]));
      }
    for (int k = (kSteps * 32 + lane) * 4; k < K; k += 128) {
#pragma unroll
      for (int e = 0; e < 4; ++e) m = max(m, abs_bits(value(k + e)));
    }
    m = __reduce_max_sync(0xffffffffu, m);
    const TokenScale s = token_scale(m);
    const uint32_t keep = m >= 0x7f800000u ? 0u : 0xffffffffu;
    const auto store = [&](int k, float a, float b, float c, float d) {
      const float2 f = scaled2(make_float2(a, b), s.inverse, s.inverse), g = scaled2(make_float2(c, d), s.inverse, s.inverse);
      *reinterpret_cast<uint32_t*>(q + t * pitch + k) = low_bytes(f.x, f.y, g.x, g.y) & keep;
    };
#pragma unroll
    for (int i = 0; i < kSteps; ++i)
      if ((i * 32 + lane) * 4 < pitch) store((i * 32 + lane) * 4, v[i][0], v[i][1], v[i][2], v[i][3]);
    for (int k = (kSteps * 32 + lane) * 4; k < pitch; k += 128)
      store(k, value(k), value(k + 1), value(k + 2), value(k + 3));
    if (lane == 0) scale[t] = s.scale;
  }
}

// ------------------------------ the product on the tensor cores ------------------------------
// D[128 rows of A, bn rows of B] = A B^T in 8-bit integers with 32-bit sums
// (tcgen05.mma kind::i8), both operands K-major rows under a 128-byte swizzle.
//
// Which operand is A goes by the output's layout and by how it is stored.  Staged (y's rows are
// whole 16-byte units): the accumulator's columns lie along y's rows, so A is the tokens for rows,
// the weights for channels-first, and a lane's 128 bytes of columns are a row of a TMA store's
// box.  (The other way round, lanes along y's rows, a warp's box has rows of 64 bytes, and
// their rate was the bound: 127 us against 118 us for the product 32768 x 1024 -> 4096.)  Unstaged:
// the lanes lie along y's rows, so that direct stores of one element per lane are coalesced.
//
// Persistent, warp-specialised: warp 0 issues the TMA loads (a ring of 128-byte K
// blocks), warp 1 owns TMEM and issues the MMAs into two to four accumulators in turn, two
// groups of four warps scale and store: a tile each in turn where TMEM holds four, so that one
// tile's latencies pass under the other's, else half of every tile each.  The waits and the exit follow
// the pointwise kernels' discipline: every wait is bounded, and what is in flight is waited for before TMEM is freed.
constexpr int kI8BM = 128, kI8BK = 128;
constexpr int kI8Threads = 320, kI8EpiWarps = 8;
constexpr int kI8MaxStages = 8, kI8MaxAcc = 4;

struct I8GemmArgs {
  const float* a_scale;  // of A's rows
  const float* b_scale;  // of B's rows
  const float* bias;     // of the output channels, or NULL
  void* y;
  int a_rows, b_rows, K;  // of one sample, where they are tokens
  int N;                  // output channels
  int bn, stages, accs;
  int share;  // the two groups share each tile
  int groups, copies;  // of quantising warps, of the channels in operand A (the medium form)
  int a_tiles, b_tiles, samples;  // tiles of one sample
};

// The tile that a CTA (or pair) takes in its turn: neighbours share a tile of tokens and
// differ in the output channels.
struct I8Tile {
  int sample, ta, tb;
};
template <bool TOKENS_A>
__device__ __forceinline__ I8Tile i8_tile(const I8GemmArgs& p, int t) {
  const int chans = TOKENS_A ? p.b_tiles : p.a_tiles, tokens = TOKENS_A ? p.a_tiles : p.b_tiles;
  const int tok = t / chans, ch = t - tok * chans, sample = tok / tokens, tt = tok - sample * tokens;
  return TOKENS_A ? I8Tile{sample, tt, ch} : I8Tile{sample, ch, tt};
}

// A staging buffer: an epilogue warp's 32 lanes, 128 bytes each (128-byte swizzle).
constexpr int kI8StageBytes = 32 * 128;

// Where a loop stands in a ring: counted, since a division by a runtime number of slots costs
// more than the K block's products.
struct RingAt {
  int slot = 0;
  uint32_t turn = 0;  // its lowest bit: the parity of the slot's current phase
  __device__ __forceinline__ void next(int slots) {
    if (++slot == slots) {
      slot = 0;
      ++turn;
    }
  }
};

struct I8Shared {
  uint64_t full[kI8MaxStages], empty[kI8MaxStages];
  uint64_t tfull[kI8MaxAcc], tempty[kI8MaxAcc];
  uint64_t drain;
  uint32_t tmem_base;
  int abort;
  float4 col[kI8EpiWarps][32];  // (scale, bias) of an epilogue warp's columns
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

// The scaling and staged store of one warp's 32 accumulator lanes of a tile, 128 bytes of
// columns at a time.
template <typename T, bool TOKENS_A>
struct StagedTile {
  static constexpr int kCols = 128 / (int)sizeof(T);
  const I8GemmArgs& p;
  float4* col;  // the warp's [kCols / 2]: two columns' scales, and biases where they are output channels
  int lane, r0, sample, b0;
  float scale, bias;  // of the lane's row

  // the constants of kCols columns: two per lane (kCols = 64) or one of each pair's lanes
  __device__ __forceinline__ void columns(int c0) {
    const float* b_scale = p.b_scale + (TOKENS_A ? 0LL : (long long)sample * p.b_rows);
    const int c = b0 + c0 + 2 * lane;
    if (2 * lane >= kCols) return;
    const bool in0 = c < p.b_rows, in1 = c + 1 < p.b_rows, biased = TOKENS_A && p.bias != nullptr;
    col[lane] = make_float4(in0 ? b_scale[c] : 0.f, in1 ? b_scale[c + 1] : 0.f, in0 && biased ? p.bias[c] : 0.f,
                            in1 && biased ? p.bias[c + 1] : 0.f);
  }
  // The constants of the row and of the first columns: on their way while the product is
  // computed.
  __device__ __forceinline__ void prepare(int first) {
    const int row = r0 + lane;
    const bool in = row < p.a_rows;
    scale = in ? p.a_scale[(TOKENS_A ? (long long)sample * p.a_rows : 0LL) + row] : 0.f;
    bias = in && !TOKENS_A && p.bias != nullptr ? p.bias[row] : 0.f;
    __syncwarp();
    columns(first);
  }
  // t0: TMEM address of the warp's lanes, column 0; stg: the warp's staging buffer.
  __device__ __forceinline__ void store(const CUtensorMap* mY, uint32_t t0, int first, int next, uint8_t* stg) {
    for (int c0 = first; c0 < p.bn && b0 + c0 < p.b_rows; c0 += next) {
      __syncwarp();  // the previous piece's constants are read
      if (c0 > first) columns(c0);
      uint32_t r[kCols / 32][32];
#pragma unroll
      for (int h = 0; h < kCols / 32; ++h) tmem_ld32(t0 + (uint32_t)(c0 + 32 * h), r[h]);
      if (lane == 0) bulk_wait_read<0>();  // the last store has read the buffer
      __syncwarp();
      tmem_ld_wait();
#pragma unroll
      for (int h = 0; h < kCols / 32; ++h) {
        float2 out[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float4 k = col[16 * h + j];
          const float2 v = make_float2((float)(int)r[h][2 * j], (float)(int)r[h][2 * j + 1]);
          // (sum * token's scale) * channel's scale + bias
          out[j] = TOKENS_A ? __ffma2_rn(__fmul2_rn(v, make_float2(scale, scale)), make_float2(k.x, k.y), make_float2(k.z, k.w))
                            : __ffma2_rn(__fmul2_rn(v, make_float2(k.x, k.y)), make_float2(scale, scale), make_float2(bias, bias));
        }
        const float* f = reinterpret_cast<const float*>(out);
        constexpr int E = 16 / sizeof(T);
#pragma unroll
        for (int u = 0; u < 32 / E; ++u)
          *reinterpret_cast<uint4*>(stg + lane * 128 + (((h * (32 / E) + u) ^ (lane & 7)) << 4)) = pack16<T>(f + u * E);
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) {
        if (r0 < p.a_rows) tma_store_3d(mY, stg, b0 + c0, r0, sample);
        bulk_commit();
      }
    }
  }
};

template <typename T, bool TOKENS_A, bool STAGED>
__global__ void __launch_bounds__(kI8Threads, 1)
    i8_gemm_kernel(const __grid_constant__ CUtensorMap mA, const __grid_constant__ CUtensorMap mB,
                   const __grid_constant__ CUtensorMap mY, I8GemmArgs p) {
  extern __shared__ uint8_t i8_raw[];
  __shared__ I8Shared sh;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* ringA = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(i8_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* ringB = ringA + (size_t)p.stages * (kI8BM * kI8BK);
  const int b_bytes = p.bn * kI8BK;
  uint8_t* stage = ringB + (size_t)p.stages * b_bytes;
  const uint32_t tmem_cols = (uint32_t)(p.accs * p.bn);
  if (warp == 1) tmem_alloc(&sh.tmem_base, tmem_cols);
  if (threadIdx.x == 0) {
    for (int i = 0; i < p.stages; ++i) {
      mbar_init(&sh.full[i], 1);
      mbar_init(&sh.empty[i], 1);
    }
    for (int i = 0; i < p.accs; ++i) {
      mbar_init(&sh.tfull[i], 1);
      mbar_init(&sh.tempty[i], kI8EpiWarps * (p.share ? 32 : 16));
    }
    mbar_init(&sh.drain, 1);
    sh.abort = 0;
    fence_mbarrier_init();
    tma_prefetch_map(&mA);
    tma_prefetch_map(&mB);
    if (STAGED) tma_prefetch_map(&mY);
  }
  if (warp == 1) tmem_relinquish();
  grid_dependency_wait();  // the set-up above passes under the quantisation's end
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem_base;
  volatile int* abort = &sh.abort;
  const int tiles = p.a_tiles * p.b_tiles * p.samples;
  const int mine = (tiles - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x;
  const int kblocks = (p.K + kI8BK - 1) / kI8BK;
  long long issued = 0;
  const auto decode = [&](int i, int& sample, int& a0, int& b0) {
    const I8Tile t = i8_tile<TOKENS_A>(p, (int)blockIdx.x + i * (int)gridDim.x);
    sample = t.sample;
    a0 = t.ta * kI8BM;
    b0 = t.tb * p.bn;
  };

  if (warp == 0) {
    if (lane == 0) {
      bool ok = true;
      RingAt at;
      for (int i = 0; i < mine && ok; ++i) {
        int sample, a0, b0;
        decode(i, sample, a0, b0);
        for (int kb = 0; kb < kblocks; ++kb, at.next(p.stages)) {
          const int st = at.slot;
          if (at.turn > 0 && !(ok = wait_or_abort(&sh.empty[st], (at.turn - 1) & 1, abort))) break;
          mbar_arrive_expect_tx(&sh.full[st], (uint32_t)(kI8BM * kI8BK + b_bytes));
          tma_load_3d(ringA + (size_t)st * (kI8BM * kI8BK), &mA, &sh.full[st], kb * kI8BK, a0, TOKENS_A ? sample : 0);
          tma_load_3d(ringB + (size_t)st * b_bytes, &mB, &sh.full[st], kb * kI8BK, b0, TOKENS_A ? 0 : sample);
          ++issued;
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = make_idesc_i8(kI8BM, p.bn);
      RingAt at;
      bool ok = true;
      for (int i = 0; i < mine && ok; ++i) {
        const int acc = i % p.accs, turn = i / p.accs;
        if (turn > 0 && !wait_or_abort(&sh.tempty[acc], (uint32_t)((turn - 1) & 1), abort)) break;
        tc_fence_after();
        const uint32_t d = tmem + (uint32_t)(acc * p.bn);
        for (int kb = 0; kb < kblocks; ++kb, at.next(p.stages)) {
          const int st = at.slot;
          if (!(ok = wait_or_abort(&sh.full[st], at.turn & 1, abort))) break;
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
    // accumulator lanes 32 * (warp % 4) ..; 128 bytes or 32 columns at a time
    const int q4 = warp & 3, half = (warp - 2) >> 2;
    constexpr int kPiece = STAGED ? 128 / (int)sizeof(T) : 32;
    const int first = p.share ? half * kPiece : 0, next = p.share ? 2 * kPiece : kPiece;
    float2* col = reinterpret_cast<float2*>(sh.col[warp - 2]);
    uint8_t* stg = stage + (warp - 2) * kI8StageBytes;
    for (int i = p.share ? 0 : half; i < mine; i += p.share ? 1 : 2) {
      const int acc = i % p.accs;
      int sample, a0, b0;
      decode(i, sample, a0, b0);
      const int r0 = a0 + q4 * 32;  // this warp's first row of A
      // (false: a wait ran out, the warp leaves)
      const auto accumulated = [&] {
        if (!__all_sync(0xffffffffu, wait_or_abort(&sh.tfull[acc], (uint32_t)((i / p.accs) & 1), abort))) return false;
        tc_fence_after();
        return true;
      };
      const uint32_t t0 = tmem + (uint32_t)(acc * p.bn) + ((uint32_t)(q4 * 32) << 16);
      if constexpr (STAGED) {
        StagedTile<T, TOKENS_A> tile{p, sh.col[warp - 2], lane, r0, sample, b0, 0.f, 0.f};
        tile.prepare(first);
        if (!accumulated()) break;
        tile.store(&mY, t0, first, next, stg);
      } else {
        const int row = r0 + lane;
        const bool in = row < p.a_rows;
        // TOKENS_A goes with channels-first here
        const float row_scale = in ? p.a_scale[(TOKENS_A ? (long long)sample * p.a_rows : 0LL) + row] : 0.f;
        const float row_bias = !TOKENS_A && in && p.bias != nullptr ? p.bias[row] : 0.f;
        const long long step = TOKENS_A ? p.a_rows : p.N;  // of y, from one column to the next
        T* y = static_cast<T*>(p.y) + row +
               (TOKENS_A ? ((long long)sample * p.N + b0) * p.a_rows : (long long)b0 * p.N);
        if (!accumulated()) break;
        for (int c0 = first; c0 < p.bn && b0 + c0 < p.b_rows; c0 += next) {
          uint32_t r[32];
          __syncwarp();  // whole again, and the previous piece's constants are read
          tmem_ld32(t0 + (uint32_t)c0, r);
          const int c = b0 + c0 + lane;
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
            if (in && j < n)
              *at = from_acc<T>(TOKENS_A ? fmaf(v * row_scale, k.x, k.y) : fmaf(v * k.x, row_scale, row_bias));
            at += step;
          }
        }
      }
      __syncwarp();
      tc_fence_before();
      mbar_arrive(&sh.tempty[acc]);
    }
    if (STAGED && lane == 0) bulk_wait_all();
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

// ------------------------------ large products: two SMs per tile ------------------------------
// One SM's 128 x 256 tile takes 48 KB of operands per 128 of K through the SM's load port, more
// than the port's share of the tensor core's time (at 64 bytes a clock 768 clocks against 512).
// A pair of CTAs (a cluster, tcgen05 cta_group::2) computes 256 x 256: each loads its 128 rows
// of A and 128 of B's 256 rows, 32 KB, and the instruction reads both halves of B.
//
// The even CTA leads: its warp 1 issues the MMAs for both, whose accumulators lie in each
// CTA's own TMEM.  Both CTAs' loads complete on the leader's barriers; a commit releases the
// slot in both.  Epilogue warps of both release an accumulator at the leader.  The rest is as in the
// kernel above; an accumulator is drained by all eight warps of its CTA.
//
// 8192 x 4096 -> 4096 bf16: 98 us in the product, 2.8 POP/s (one SM per tile: 131 us);
// 32768 x 1024 -> 4096: 118 us, 2.3 POP/s, the epilogue and its 268 MB of output sharing the
// bound.
constexpr int kI8PairStages = 5;

__device__ __forceinline__ uint32_t cluster_addr(const void* p, uint32_t rank) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
// A load into this CTA that completes on a barrier of the pair's leader.
__device__ __forceinline__ void tma_load_3d_pair(void* dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 "
      "[%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
__device__ __forceinline__ void mma_i8_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Arrives at the same barrier of both CTAs once the MMAs issued so far are done.
__device__ __forceinline__ void mma_commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}

template <typename T, bool TOKENS_A>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kI8Threads, 1)
    i8_gemm_pair_kernel(const __grid_constant__ CUtensorMap mA, const __grid_constant__ CUtensorMap mB,
                        const __grid_constant__ CUtensorMap mY, I8GemmArgs p) {
  extern __shared__ uint8_t i8_raw[];
  __shared__ I8Shared sh;
  constexpr int kHalf = kI8BM * kI8BK, kAccs = 2, kCols = 512;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)(blockIdx.x & 1);  // the cluster's CTAs are neighbours
  uint8_t* ringA = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(i8_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* ringB = ringA + (size_t)kI8PairStages * kHalf;
  uint8_t* stage = ringB + (size_t)kI8PairStages * kHalf;
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem_base)),
                 "r"((uint32_t)kCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < kI8PairStages; ++i) {
      mbar_init(&sh.full[i], 1);
      mbar_init(&sh.empty[i], 1);
    }
    for (int i = 0; i < kAccs; ++i) {
      mbar_init(&sh.tfull[i], 1);
      mbar_init(&sh.tempty[i], 2 * kI8EpiWarps);
    }
    mbar_init(&sh.drain, 1);
    sh.abort = 0;
    fence_mbarrier_init();
    tma_prefetch_map(&mA);
    tma_prefetch_map(&mB);
    tma_prefetch_map(&mY);
  }
  grid_dependency_wait();
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // the pair's barriers are there
  tc_fence_after();
  const uint32_t tmem = sh.tmem_base;
  volatile int* abort = &sh.abort;
  const int tiles = p.a_tiles * p.b_tiles * p.samples;
  const int pair = (int)(blockIdx.x >> 1), pairs = (int)(gridDim.x >> 1);
  const int mine = (tiles - pair + pairs - 1) / pairs;
  const int kblocks = (p.K + kI8BK - 1) / kI8BK;
  long long issued = 0;
  const auto decode = [&](int i, int& sample, int& a0, int& b0) {  // a0: of this CTA's rows
    const I8Tile t = i8_tile<TOKENS_A>(p, pair + i * pairs);
    sample = t.sample;
    a0 = t.ta * (2 * kI8BM) + rank * kI8BM;
    b0 = t.tb * 256;
  };

  if (warp == 0) {
    if (lane == 0) {
      bool ok = true;
      RingAt at;
      for (int i = 0; i < mine && ok; ++i) {
        int sample, a0, b0;
        decode(i, sample, a0, b0);
        for (int kb = 0; kb < kblocks; ++kb, at.next(kI8PairStages)) {
          const int st = at.slot;
          if (at.turn > 0 && !(ok = wait_or_abort(&sh.empty[st], (at.turn - 1) & 1, abort))) break;
          if (rank == 0) mbar_arrive_expect_tx(&sh.full[st], 4 * kHalf);  // both CTAs' bytes
          const uint32_t bar = cluster_addr(&sh.full[st], 0);
          tma_load_3d_pair(ringA + (size_t)st * kHalf, &mA, bar, kb * kI8BK, a0, TOKENS_A ? sample : 0);
          tma_load_3d_pair(ringB + (size_t)st * kHalf, &mB, bar, kb * kI8BK, b0 + rank * kI8BM, TOKENS_A ? 0 : sample);
          ++issued;
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      const uint32_t idesc = make_idesc_i8(2 * kI8BM, 256);
      RingAt at;
      bool ok = true;
      for (int i = 0; i < mine && ok; ++i) {
        const int acc = i % kAccs, turn = i / kAccs;
        if (turn > 0 && !wait_or_abort(&sh.tempty[acc], (uint32_t)((turn - 1) & 1), abort)) break;
        tc_fence_after();
        const uint32_t d = tmem + (uint32_t)(acc * 256);
        for (int kb = 0; kb < kblocks; ++kb, at.next(kI8PairStages)) {
          const int st = at.slot;
          if (!(ok = wait_or_abort(&sh.full[st], at.turn & 1, abort))) break;
          tc_fence_after();
          const uint32_t sa = smem_u32(ringA + (size_t)st * kHalf), sb = smem_u32(ringB + (size_t)st * kHalf);
          const int steps = min(kI8BK, p.K - kb * kI8BK + 31) / 32;
          for (int ks = 0; ks < steps; ++ks)
            mma_i8_pair(d, make_sw128_desc(sa + ks * 32, 16, 1024), make_sw128_desc(sb + ks * 32, 16, 1024), idesc,
                        kb > 0 || ks > 0 ? 1u : 0u);
          mma_commit_pair(&sh.empty[st]);
        }
        if (ok) mma_commit_pair(&sh.tfull[acc]);
      }
    }
  } else {
    const int q4 = warp & 3, half = (warp - 2) >> 2;
    constexpr int kPiece = 128 / (int)sizeof(T);
    uint8_t* stg = stage + (warp - 2) * kI8StageBytes;
    for (int i = 0; i < mine; ++i) {
      const int acc = i % kAccs;
      int sample, a0, b0;
      decode(i, sample, a0, b0);
      StagedTile<T, TOKENS_A> tile{p, sh.col[warp - 2], lane, a0 + q4 * 32, sample, b0, 0.f, 0.f};
      tile.prepare(half * kPiece);
      if (!__all_sync(0xffffffffu, wait_or_abort(&sh.tfull[acc], (uint32_t)((i / kAccs) & 1), abort))) break;
      tc_fence_after();
      tile.store(&mY, tmem + (uint32_t)(acc * 256) + ((uint32_t)(q4 * 32) << 16), half * kPiece, 2 * kPiece, stg);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(cluster_addr(&sh.tempty[acc], 0));
    }
    if (lane == 0) bulk_wait_all();
  }
  __syncthreads();
  if (*abort && lane == 0 && rank == 0) {
    if (warp == 0) drain_ring(sh.full, kI8PairStages, issued);
    if (warp == 1) {
      mma_commit_pair(&sh.drain);
      mbar_wait(&sh.drain, 0);
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // neither CTA's memory is in use by the other any more
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)kCols) : "memory");
}

// ------------------------------ narrow products in one kernel ------------------------------
// Channels first with weights that stay in shared memory: the product is bound by the
// bytes of x and y, so x is read, quantised, multiplied and written by the same CTA, and
// no 8-bit rows go through memory (the two-kernel form reads and writes K bytes per token
// more, and its accumulators pass through TMEM: 248 us against this kernel's 84 us for
// 32 -> 64 channels at 128^3, where x and y take 62 us of bandwidth).
//
// A tile is 32 W tokens.  Warp s of S = ceil(K / 32) quantises channels 32 s .. of it as
// i8_quantize_chan_kernel does, into token rows in shared memory.  Then the warps share the
// output channels, 16 at a time: mma.sync m16n8k32 with the weights as A, so that sums stay
// in the registers of the thread that stores them.  Column n of the four B fragments of 32
// tokens is token 8 (n / 2) + 2 j + n % 2 of them: a thread's columns 2 t, 2 t + 1 of
// fragments j = 0 .. 3 are 8 neighbouring tokens, 16 bytes of 16-bit data.  A warp's
// channels (up to 64) x the tile's 128 bytes of tokens go through shared memory and leave in
// one TMA store where y's rows are whole 16-byte units: stored directly, a warp's 16-byte pieces
// in 8 rows keep the L1 data pipe busy (74 %, the bound), and in many small TMA stores (16
// channels x 64 bytes) their issue is the bound.
__device__ __forceinline__ void mma_s8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

struct I8NarrowArgs {
  const void* x;
  const int8_t* w;
  const float* ws;
  const float* bias;  // or NULL
  void* y;
  long long w_pitch;
  int outer, inner, K, N;
  int mt_warp, mt_store;  // 16-channel pieces per warp, and per store (a divisor)
};

// Shared memory: a staging buffer per warp, weights [N16][row], per output channel (scale,
// bias), then per tile of the CTA: token rows [32 W][row], their scales, and the warps' maxima
// [S][W][32].  row = K
// rounded up to 32, plus 16: an odd number of 16-byte units, so that eight neighbouring rows'
// ldmatrix reads fall on different banks; eight tokens' rows take 32 bytes more, which does
// the same for the permuted tokens of a B fragment.
__host__ __device__ __forceinline__ int narrow_row(int K) { return (K + 31) / 32 * 32 + 16; }
__host__ __device__ __forceinline__ int narrow_token(int t, int row) { return t * row + (t >> 3) * 32; }
__host__ __device__ __forceinline__ int narrow_tile_bytes(int K, int W) {
  return narrow_token(32 * W, narrow_row(K)) + 32 * W * 4 + (K + 31) / 32 * W * 128;
}
__host__ __device__ __forceinline__ int narrow_weight_bytes(int K, int N) {
  return (N + 15) / 16 * 16 * (narrow_row(K) + 8);
}

// Bytes of staging per 16 channels: 128-byte rows (64 tokens of 16-bit data, 32 of fp32),
// 128-byte swizzle.
constexpr int kNarrowStage = 16 * 128;
constexpr int kNarrowMtStore = 2;
constexpr int kNarrowWarps = 16;  // resident per SM, at 128 registers
template <typename T>
constexpr int kNarrowW = 4 / (int)sizeof(T);  // tokens per lane

// S = KB = ceil(K / 32) is 1 or 2: a tile's B fragments stay in registers over the output
// channels.  The sums are below 2^22, so they start from the bits of 1.5 * 2^23 and are the
// mantissa of a float already: a subtraction takes the place of the conversion, which runs
// at an eighth of the rate.
constexpr int kSumBits = 0x4B400000;

template <typename T, int KB>
__global__ void __launch_bounds__(kNarrowWarps * 32, 1)
    i8_narrow_kernel(const __grid_constant__ CUtensorMap mY, I8NarrowArgs a) {
  constexpr int W = kNarrowW<T>, S = KB;
  extern __shared__ uint8_t i8_raw[];
  const int lane = threadIdx.x, s = threadIdx.y, P = blockDim.z;
  const int row = narrow_row(a.K), n16 = (a.N + 15) / 16;
  uint8_t* base_sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(i8_raw) + 1023) & ~(uintptr_t)1023);
  const int stage_bytes = a.mt_store * kNarrowStage;
  uint8_t* stg = base_sm + (s + S * threadIdx.z) * stage_bytes;
  uint8_t* wsm = base_sm + S * P * stage_bytes;
  float2* chan = reinterpret_cast<float2*>(wsm + n16 * 16 * row);
  uint8_t* tile_sm = wsm + narrow_weight_bytes(a.K, a.N) + threadIdx.z * narrow_tile_bytes(a.K, W);
  float* tscale = reinterpret_cast<float*>(tile_sm + narrow_token(32 * W, row));
  uint32_t* maxima = reinterpret_cast<uint32_t*>(tscale + 32 * W);
  {
    const int me = threadIdx.x + 32 * (threadIdx.y + S * threadIdx.z), all = 32 * S * P;
    for (int i = me; i < n16 * 16 * 2 * KB; i += all) {
      const int n = i / (2 * KB), k = (i - n * (2 * KB)) * 16;
      uint4 v = make_uint4(0, 0, 0, 0);
      // the last 16 bytes of a row may hold bytes past K: they meet zeros of x
      if (n < a.N && k < a.K) v = *reinterpret_cast<const uint4*>(a.w + n * a.w_pitch + k);
      *reinterpret_cast<uint4*>(wsm + n * row + k) = v;
    }
    for (int n = me; n < n16 * 16; n += all)
      chan[n] = n < a.N ? make_float2(a.ws[n], a.bias != nullptr ? a.bias[n] : 0.f) : make_float2(0.f, 0.f);
  }
  __syncthreads();
  // the warps of a tile meet at a barrier of their own
  const auto meet = [&] {
    if (S > 1) asm volatile("bar.sync %0, %1;" ::"r"((int)threadIdx.z + 1), "n"(32 * S) : "memory");
    else __syncwarp();
  };
  const int per = (a.inner + 32 * W - 1) / (32 * W);
  const long long tiles = (long long)a.outer * per;
  const uint32_t w_addr = smem_u32(wsm), t_addr = smem_u32(tile_sm);
  const int g = lane >> 2, t4 = lane & 3;
  // ldmatrix row addresses: A takes rows 0-7, 8-15 of the first 16 bytes, then of the second;
  // B takes fragment j's two halves, then fragment j + 1's, rows being the permuted tokens
  const uint32_t a_off = (uint32_t)((lane & 15) * row + (lane >> 4) * 16);
  const int bn = lane & 7;
  const uint32_t b_off = (uint32_t)(narrow_token(8 * (bn >> 1) + 2 * (lane >> 4) + (bn & 1), row) + ((lane >> 3) & 1) * 16);
  const int mine = min(32, a.K - s * 32), mt_end = min(n16, (s + 1) * a.mt_warp);
  uint32_t x[32];
  // the tile's x: of the first before the loop, of each next one as soon as the last is
  // quantised, so that its loads pass under the products and the stores
  const auto load = [&](long long tile) {
    const int o = (int)(tile / per), v = (int)(tile - (long long)o * per) * (32 * W) + lane * W;
    const bool in = tile < tiles && v < a.inner;  // inner is a multiple of W
    const T* px = static_cast<const T*>(a.x) + ((long long)o * a.K + s * 32) * a.inner + v;
#pragma unroll
    for (int k = 0; k < 32; ++k) {
      x[k] = in && k < mine ? *reinterpret_cast<const uint32_t*>(px) : 0u;
      px += a.inner;
      asm volatile("" : "+l"(px));  // one address in flight, not 32
    }
  };
  load((long long)blockIdx.x * P + threadIdx.z);
  for (long long base = (long long)blockIdx.x * P; base < tiles; base += (long long)gridDim.x * P) {
    const long long tile = base + threadIdx.z;
    const int o = (int)(tile / per), v0 = (int)(tile - (long long)o * per) * (32 * W);
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < 32; ++k) m = W == 2 ? __vmaxu2(m, x[k] & 0x7fff7fffu) : max(m, x[k] & 0x7fffffffu);
    uint32_t most[W];
    if constexpr (W == 2) {
      most[0] = Mag<T>::lo(m);
      most[1] = Mag<T>::hi(m);
    } else {
      most[0] = m;
    }
    if (S > 1) {
#pragma unroll
      for (int j = 0; j < W; ++j) maxima[(s * W + j) * 32 + lane] = most[j];
    }
    meet();  // the maxima are there, and the last tile's rows are read
    if (S > 1) {
#pragma unroll
      for (int j = 0; j < W; ++j) most[j] = max(maxima[j * 32 + lane], maxima[(W + j) * 32 + lane]);
    }
    TokenScale ts[W];
#pragma unroll
    for (int j = 0; j < W; ++j) {
      ts[j] = token_scale(most[j]);
      if (s == 0) tscale[lane * W + j] = ts[j].scale;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t b[W][4];
      quantize16<T, W>(x + h * 16, ts, b);
#pragma unroll
      for (int j = 0; j < W; ++j) {
        const uint32_t keep = most[j] >= 0x7f800000u ? 0u : 0xffffffffu;
        *reinterpret_cast<uint4*>(tile_sm + narrow_token(lane * W + j, row) + s * 32 + h * 16) =
            make_uint4(b[j][0] & keep, b[j][1] & keep, b[j][2] & keep, b[j][3] & keep);
      }
    }
    meet();
    if (base + (long long)gridDim.x * P < tiles) load(tile + (long long)gridDim.x * P);
#pragma unroll 1
    for (int mt0 = s * a.mt_warp; tile < tiles && mt0 < mt_end; mt0 += a.mt_store) {
      if (lane == 0) bulk_wait_read<0>();  // the last store has read the buffer
      __syncwarp();
#pragma unroll 1
      for (int part = 0; part < W; ++part) {  // 32 tokens at a time
        const int tok = part * 32 + 8 * t4;
        const uint32_t b_addr = t_addr + (uint32_t)narrow_token(part * 32, row) + b_off;
        const float4 lo = *reinterpret_cast<const float4*>(tscale + tok);
        const float4 hi = *reinterpret_cast<const float4*>(tscale + tok + 4);
        const float2 sc[4] = {make_float2(lo.x, lo.y), make_float2(lo.z, lo.w), make_float2(hi.x, hi.y),
                              make_float2(hi.z, hi.w)};
        uint32_t fb[KB][2][4];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          ldsm_x4(b_addr + kb * 32, fb[kb][0]);
          ldsm_x4(b_addr + (uint32_t)(4 * row) + kb * 32, fb[kb][1]);
        }
#pragma unroll 1
        for (int mt = mt0; mt < min(mt_end, mt0 + a.mt_store); ++mt) {
          int acc[4][4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[j][i] = kSumBits;
          const uint32_t a_addr = w_addr + (uint32_t)(mt * 16 * row) + a_off;
#pragma unroll
          for (int kb = 0; kb < KB; ++kb) {
            uint32_t fa[4];
            ldsm_x4(a_addr + kb * 32, fa);
#pragma unroll
            for (int j = 0; j < 4; ++j) mma_s8(acc[j], fa, fb[kb][j >> 1][(j & 1) * 2], fb[kb][j >> 1][(j & 1) * 2 + 1]);
          }
          uint8_t* buf = stg + (mt - mt0) * kNarrowStage;
#pragma unroll
          for (int h = 0; h < 2; ++h) {  // channels g and g + 8
            const int r = h * 8 + g;
            const float2 c = chan[mt * 16 + r];  // zeros past N
            float2 out[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float2 v = __fadd2_rn(make_float2(__int_as_float(acc[j][h * 2]), __int_as_float(acc[j][h * 2 + 1])),
                                          make_float2(-kRint, -kRint));
              out[j] = __ffma2_rn(__fmul2_rn(v, sc[j]), make_float2(c.x, c.x), make_float2(c.y, c.y));
            }
            const float* f = reinterpret_cast<const float*>(out);
            if constexpr (W == 2) {
              *reinterpret_cast<uint4*>(buf + r * 128 + (((part * 4 + t4) ^ (r & 7)) << 4)) = pack16<T>(f);
            } else {
              *reinterpret_cast<uint4*>(buf + r * 128 + (((2 * t4) ^ (r & 7)) << 4)) = pack16<T>(f);
              *reinterpret_cast<uint4*>(buf + r * 128 + (((2 * t4 + 1) ^ (r & 7)) << 4)) = pack16<T>(f + 4);
            }
          }
        }
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) {
        tma_store_3d(&mY, stg, v0, mt0 * 16, o);
        bulk_commit();
      }
    }
  }
  if (lane == 0) bulk_wait_all();
}

// 16-channel pieces per warp and per store: the most, up to kNarrowMtStore, that divide a warp's share
// (a store's box may not reach into the next warp's channels).
void narrow_share(int N, int S, int* mt_warp, int* mt_store) {
  *mt_warp = ((N + 15) / 16 + S - 1) / S;
  *mt_store = kNarrowMtStore;
  while (*mt_warp % *mt_store != 0) --*mt_store;
}
// Shared memory of a CTA of P tiles.
size_t narrow_smem(int K, int N, int W, int P) {
  const int S = (K + 31) / 32;
  int mt_warp, mt_store;
  narrow_share(N, S, &mt_warp, &mt_store);
  return (size_t)narrow_weight_bytes(K, N) + (size_t)P * (narrow_tile_bytes(K, W) + S * mt_store * kNarrowStage) + 1024;
}
// Whether the one-kernel form takes a product: K and N small enough that bytes are its bound
// (bf16, 64^3 voxels: 64 -> 192 channels 42 us against 51 us in two kernels; wider ones go to the
// medium form), whole 16-byte rows, and enough tiles.
bool narrow_takes(const void* x, const void* y, long long outer, int K, long long inner, int N, size_t esz) {
  return K <= 64 && N <= 256 && inner % (16 / (long long)esz) == 0 && reinterpret_cast<uintptr_t>(x) % 4 == 0 &&
         reinterpret_cast<uintptr_t>(y) % 16 == 0 && outer * ((inner + 63) / 64) >= 2 * kI8Sms;
}

// ------------------------------ a few tokens ------------------------------
// Up to eight tokens: the weights' bytes and the launch count, not the tokens.  One kernel:
// a warp owns one output channel and asks for the first 2 KB of its weights before anything
// else; meanwhile the CTA quantises all tokens into shared memory (each CTA for itself: they
// are a few KB, from L2).  Then dot products of four bytes a lane, and a warp sum.
// One token 512 -> 2048: 3.9 us; as two kernels 8.3 us.
constexpr int kI8FewTokens = 8, kI8FewWarps = 8;

struct I8FewArgs {
  const void* x;
  const int8_t* w;
  const float* ws;
  const float* bias;  // or NULL
  void* y;
  long long w_pitch;
  int tokens, inner, K, N;
  int per_token;  // warps that quantise a token
};

template <typename T>
__global__ void __launch_bounds__(kI8FewWarps * 32) i8_few_kernel(I8FewArgs a) {
  extern __shared__ __align__(16) uint8_t i8_few[];  // [tokens][K rounded up to 16]
  __shared__ uint32_t most[kI8FewWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n = blockIdx.x * kI8FewWarps + warp;
  const int row = (a.K + 15) / 16 * 16, chunks = row / 16;
  const uint4* w = reinterpret_cast<const uint4*>(a.w + (long long)n * a.w_pitch);
  uint4 ahead[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    ahead[i] = n < a.N && lane + 32 * i < chunks ? w[lane + 32 * i] : make_uint4(0, 0, 0, 0);
  // four values per lane and turn
  const int token = warp / a.per_token, part = warp - token * a.per_token;
  const int o = token / a.inner;
  const T* x = static_cast<const T*>(a.x) + (long long)o * a.K * a.inner + (token - o * a.inner);
  const auto value = [&](int k) { return k < a.K ? to_acc<T>(x[(long long)k * a.inner]) : 0.f; };
  uint32_t m = 0;
  if (token < a.tokens)
    for (int k = (part * 32 + lane) * 4; k < a.K; k += a.per_token * 128) {
#pragma unroll
      for (int e = 0; e < 4; ++e) m = max(m, abs_bits(value(k + e)));
    }
  m = __reduce_max_sync(0xffffffffu, m);
  if (lane == 0) most[warp] = m;
  __syncthreads();
  if (token < a.tokens) {
    for (int i = 0; i < a.per_token; ++i) m = max(m, most[token * a.per_token + i]);
    const TokenScale ts = token_scale(m);
    const uint32_t keep = m >= 0x7f800000u ? 0u : 0xffffffffu;
    for (int k = (part * 32 + lane) * 4; k < row; k += a.per_token * 128) {
      const float2 f = scaled2(make_float2(value(k), value(k + 1)), ts.inverse, ts.inverse);
      const float2 g = scaled2(make_float2(value(k + 2), value(k + 3)), ts.inverse, ts.inverse);
      *reinterpret_cast<uint32_t*>(i8_few + token * row + k) = low_bytes(f.x, f.y, g.x, g.y) & keep;
    }
  }
  __syncthreads();
  if (n >= a.N) return;
  int acc[kI8FewTokens] = {};
  const auto dot = [&](const uint4& v, int c) {
#pragma unroll
    for (int t = 0; t < kI8FewTokens; ++t) {
      if (t >= a.tokens) break;
      const uint4 u = *reinterpret_cast<const uint4*>(i8_few + t * row + c * 16);
      acc[t] = __dp4a((int)v.x, (int)u.x, acc[t]);
      acc[t] = __dp4a((int)v.y, (int)u.y, acc[t]);
      acc[t] = __dp4a((int)v.z, (int)u.z, acc[t]);
      acc[t] = __dp4a((int)v.w, (int)u.w, acc[t]);
    }
  };
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (lane + 32 * i < chunks) dot(ahead[i], lane + 32 * i);
  for (int c = lane + 128; c < chunks; c += 32) dot(w[c], c);
  const float scale = a.ws[n], bias = a.bias != nullptr ? a.bias[n] : 0.f;
#pragma unroll
  for (int t = 0; t < kI8FewTokens; ++t) {
    if (t >= a.tokens) break;
    const int sum = __reduce_add_sync(0xffffffffu, acc[t]);
    if (lane == t) {
      uint32_t mt = 0;
      for (int i = 0; i < a.per_token; ++i) mt = max(mt, most[t * a.per_token + i]);
      const int ot = t / a.inner;
      static_cast<T*>(a.y)[((long long)ot * a.N + n) * a.inner + (t - ot * a.inner)] =
          from_acc<T>(fmaf((float)sum * token_scale(mt).scale, scale, bias));
    }
  }
}

// Whether the one-kernel form for a few tokens takes a product: its 8-bit rows fit.
bool few_takes(long long tokens, int K) { return tokens <= kI8FewTokens && tokens * ((K + 15) / 16 * 16) <= 64 * 1024; }

template <typename T>
int launch_few(I8FewArgs a, cudaStream_t s) {
  int tokens = 1;
  while (tokens < a.tokens) tokens *= 2;
  a.per_token = kI8FewWarps / tokens;
  const size_t smem = (size_t)a.tokens * ((a.K + 15) / 16 * 16);
  const int st = ensure_smem(i8_few_kernel<T>, smem);
  if (st != MEDNEXT_OK) return st;
  i8_few_kernel<T><<<(a.N + kI8FewWarps - 1) / kI8FewWarps, kI8FewWarps * 32, smem, s>>>(a);
  return record_launch();
}

// ------------------------------ few hundred tokens: one cluster per tile ------------------------------
// A few hundred tokens are too few 128-row tiles for the SMs, and a long K is a long chain of
// loads in each of them: 2048 -> 512 channels at 8^3 are 32 CTAs of 16 K blocks, which an SM takes
// in at about 60 GB/s.  Here a cluster of S CTAs takes 32 tokens and up to 256 output channels,
// and its CTAs share K: each quantises its slice of the tokens into shared memory, as
// operand B, and multiplies it with its slice of the weights (operand A, by TMA, under way while
// x is read).  Two things cross the cluster, through distributed shared memory: a token's
// maximum, and the integer sums, of which each CTA joins and stores 1 / S.  Maxima and integer
// sums have no order, so the bits equal the other forms'.
constexpr int kI8ClTokens = 32, kI8ClWorkers = 256, kI8ClPiece = 256;  // channels of a turn of the workers
constexpr int kI8ClHeld = 2;  // turns whose values stay in registers: x is read once up to slices of 512 channels
constexpr int kI8ClMt = 2, kI8ClSlice = 16, kI8ClStages = 8;
constexpr int kI8ClRow = 36, kI8ClCol = 132;  // words between partial sums' rows: 16-byte rows without bank conflicts

struct I8ClusterArgs {
  const void* x;
  const float* ws;
  const float* bias;  // or NULL
  void* y;
  int inner, tokens;  // tokens of a sample
  int tiles;          // tiles of a sample
  int K, N;
  int S, slice;       // CTAs of a cluster, 128-byte K blocks of a CTA
  int mt, groups;     // tiles of 128 output channels per cluster, clusters per token tile
  int stages;
  int region;         // bytes of the weights' ring, later the partial sums
  int vec_x, vec_y;   // 16-byte accesses
};

struct I8ClusterShared {
  uint64_t full[kI8ClStages], empty[kI8ClStages];
  uint64_t quantised, sums, drain;
  uint32_t tmem_base;
  int abort;
  uint32_t most[kI8ClTokens];  // of this CTA's slice
  float scale[kI8ClTokens];
};

__device__ __forceinline__ uint32_t peer_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ int4 peer_int4(uint32_t addr) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// W tokens per lane (channels first: 1, or 2 neighbouring 16-bit ones), W = 0: rows.
template <typename T, int W>
__global__ void __launch_bounds__(kI8Threads, 1)
    i8_cluster_kernel(const __grid_constant__ CUtensorMap mW, const __grid_constant__ I8ClusterArgs a) {
  extern __shared__ uint8_t i8_raw[];
  __shared__ I8ClusterShared sh;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(i8_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* qs = ring + a.region;  // [slice][32 tokens][128 bytes], 128-byte swizzle
  int* part = reinterpret_cast<int*>(ring);

  const int S = a.S, rank = (int)blockIdx.x % S, cluster = (int)blockIdx.x / S;
  const int group = cluster % a.groups, tile = cluster / a.groups;
  const int o = tile / a.tiles, v0 = (tile - o * a.tiles) * kI8ClTokens;  // sample and its first token
  const int kblocks = (a.K + kI8BK - 1) / kI8BK, active = (kblocks + a.slice - 1) / a.slice;
  const int kb0 = rank * a.slice, nkb = max(0, min(a.slice, kblocks - kb0));
  const int n0 = group * a.mt * kI8BM, mt = min(a.mt, (a.N - n0 + kI8BM - 1) / kI8BM);
  const uint32_t tmem_cols = (uint32_t)(32 * kI8ClMt);
  const int blocks = nkb * mt;  // of weights

  if (warp == 1) {
    tmem_alloc(&sh.tmem_base, tmem_cols);
    tmem_relinquish();
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < a.stages; ++i) {
      mbar_init(&sh.full[i], 1);
      mbar_init(&sh.empty[i], 1);
    }
    mbar_init(&sh.quantised, kI8ClWorkers);
    mbar_init(&sh.sums, 1);
    mbar_init(&sh.drain, 1);
    sh.abort = 0;
    fence_mbarrier_init();
    tma_prefetch_map(&mW);
  }
  if (threadIdx.x < kI8ClTokens) sh.most[threadIdx.x] = 0;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem_base;
  volatile int* abort = &sh.abort;
  int issued = 0;
  RingAt at{}, block{};  // block: tile of channels (slot) and K block (turn)
  const auto issue = [&](int end) {  // weight blocks up to end
    for (; issued < end; ++issued, at.next(a.stages), block.next(mt)) {
      const int st = at.slot, kb = (int)block.turn, m = block.slot;
      if (at.turn > 0 && !wait_or_abort(&sh.empty[st], (at.turn - 1) & 1, abort)) return;
      mbar_arrive_expect_tx(&sh.full[st], (uint32_t)(kI8BM * kI8BK));
      tma_load_3d(ring + (size_t)st * (kI8BM * kI8BK), &mW, &sh.full[st], (kb0 + kb) * kI8BK, n0 + m * kI8BM, 0);
    }
  };

  if (warp == 0) {
    if (lane == 0) issue(min(blocks, a.stages));
    __syncwarp();
    cluster_sync();  // the maxima
    if (lane == 0) issue(blocks);
  } else if (warp == 1) {
    cluster_sync();
    if (lane == 0 && nkb > 0 && wait_or_abort(&sh.quantised, 0, abort)) {
      tc_fence_after();
      constexpr uint32_t idesc = make_idesc_i8(kI8BM, kI8ClTokens);
      bool ok = true;
      for (int q = 0; q < blocks; ++q, at.next(a.stages), block.next(mt)) {
        const int st = at.slot, kb = (int)block.turn, m = block.slot;
        if (!(ok = wait_or_abort(&sh.full[st], at.turn & 1, abort))) break;
        tc_fence_after();
        const uint32_t sa = smem_u32(ring + (size_t)st * (kI8BM * kI8BK)), sb = smem_u32(qs + kb * (kI8ClTokens * kI8BK));
        const int steps = min(kI8BK, a.K - (kb0 + kb) * kI8BK + 31) / 32;  // zeros past K
        for (int ks = 0; ks < steps; ++ks)
          mma_i8_ss(tmem + (uint32_t)(m * kI8ClTokens), make_sw128_desc(sa + ks * 32, 16, 1024),
                    make_sw128_desc(sb + ks * 32, 16, 1024), idesc, kb > 0 || ks > 0 ? 1u : 0u);
        mma_commit(&sh.empty[st]);
      }
      if (ok) mma_commit(&sh.sums);
    }
    __syncwarp();
  } else {
    const int wk = warp - 2;
    const int k0 = kb0 * kI8BK, kq = k0 + nkb * kI8BK, kend = min(a.K, kq);  // quantised, and there to read
    const int pieces = (nkb * kI8BK + kI8ClPiece - 1) / kI8ClPiece;
    const T* x = static_cast<const T*>(a.x);
    // 16 bytes of a token's row of operand B
    const auto slot = [&](int token, int c) {
      const int k = c - k0;
      return qs + (k / kI8BK) * (kI8ClTokens * kI8BK) + token * kI8BK + (((k % kI8BK / 16) ^ (token & 7)) << 4);
    };
    if constexpr (W > 0) {
      // lanes along the tokens, a warp has 32 channels of a piece
      constexpr int TX = 32 / W, CH = 32 / W;
      const int tx = lane % TX, cy = lane / TX, v = v0 + tx * W;
      const bool in = v < a.inner;  // inner is even where W = 2
      const T* px = x + (long long)o * a.K * a.inner + v;
      uint32_t held[kI8ClHeld][CH];
      const auto load = [&](uint32_t (&w)[CH], int piece) {
#pragma unroll
        for (int k = 0; k < CH; ++k) {
          const int c = k0 + piece * kI8ClPiece + wk * 32 + cy * CH + k;
          const bool ok = in && c < kend;
          const T* p = px + (long long)c * a.inner;
          if constexpr (W == 2) w[k] = ok ? *reinterpret_cast<const uint32_t*>(p) : 0u;
          else if constexpr (sizeof(T) == 4) w[k] = ok ? __float_as_uint(*p) : 0u;
          else w[k] = ok ? (uint32_t)*reinterpret_cast<const uint16_t*>(p) : 0u;
        }
      };
      uint32_t m = 0;
      for (int first = 0; first < pieces; first += kI8ClHeld) {
#pragma unroll
        for (int i = 0; i < kI8ClHeld; ++i) load(held[i], first + i);
#pragma unroll
        for (int i = 0; i < kI8ClHeld; ++i)
#pragma unroll
          for (int k = 0; k < CH; ++k) {
            if constexpr (W == 2) m = __vmaxu2(m, held[i][k] & 0x7fff7fffu);
            else m = max(m, held[i][k] & (sizeof(T) == 4 ? 0x7fffffffu : 0x7fffu));
          }
      }
      uint32_t most[W];
      if constexpr (W == 2) {
        m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, TX));
        most[0] = Mag<T>::lo(m);
        most[1] = Mag<T>::hi(m);
      } else if constexpr (sizeof(T) == 4) {
        most[0] = m;
      } else {
        most[0] = abs_bits(unpack2<T>(m).x);
      }
      if (cy == 0) {
#pragma unroll
        for (int j = 0; j < W; ++j) atomicMax(&sh.most[tx * W + j], most[j]);
      }
      __syncwarp();
      cluster_sync();
#pragma unroll
      for (int j = 0; j < W; ++j) most[j] = 0;
      for (int r = 0; r < active; ++r) {
        const uint32_t at = cluster_addr(&sh.most[tx * W], (uint32_t)r);
#pragma unroll
        for (int j = 0; j < W; ++j) most[j] = max(most[j], peer_u32(at + 4 * j));
      }
      TokenScale ts[W];
#pragma unroll
      for (int j = 0; j < W; ++j) ts[j] = token_scale(most[j]);
      if (wk == 0 && cy == 0) {
#pragma unroll
        for (int j = 0; j < W; ++j) sh.scale[tx * W + j] = ts[j].scale;
      }
      for (int first = 0; first < pieces; first += kI8ClHeld) {
        if (pieces > kI8ClHeld) {
#pragma unroll
          for (int i = 0; i < kI8ClHeld; ++i) load(held[i], first + i);
        }
#pragma unroll
        for (int i = 0; i < kI8ClHeld; ++i)
#pragma unroll
          for (int h = 0; h < CH / 16; ++h) {
            const int c = k0 + (first + i) * kI8ClPiece + wk * 32 + cy * CH + h * 16;
            if (c >= kq) break;
            uint32_t b[W][4];
            quantize16<T, W>(held[i] + h * 16, ts, b);
#pragma unroll
            for (int j = 0; j < W; ++j) {
              const uint32_t keep = most[j] >= 0x7f800000u ? 0u : 0xffffffffu;
              *reinterpret_cast<uint4*>(slot(tx * W + j, c)) =
                  make_uint4(b[j][0] & keep, b[j][1] & keep, b[j][2] & keep, b[j][3] & keep);
            }
          }
      }
    } else {
      // a warp has four tokens, a lane 8 neighbouring values of each
      using M = Mag<T>;
      using Words = typename M::Word[4][4];
      Words held[kI8ClHeld];
      const auto load = [&](Words& w, int piece) {
        const int c = k0 + piece * kI8ClPiece + lane * 8;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const int token = v0 + wk * 4 + t;
          const T* p = x + (long long)token * a.K + c;
          if (a.vec_x) {  // K is a multiple of the vector's values
            constexpr int E = 16 / (int)sizeof(T);
#pragma unroll
            for (int h = 0; h < 8 / E; ++h) {
              const uint4 r = token < a.tokens && c + h * E < kend ? *reinterpret_cast<const uint4*>(p + h * E)
                                                                   : make_uint4(0, 0, 0, 0);
              memcpy(&w[t][h * E / 2], &r, 16);
            }
          } else {
            T e[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = token < a.tokens && c + i < kend ? p[i] : from_acc<T>(0.f);
            memcpy(w[t], e, sizeof(e));
          }
        }
      };
      typename M::Max m[4] = {};
      for (int first = 0; first < pieces; first += kI8ClHeld) {
#pragma unroll
        for (int p = 0; p < kI8ClHeld; ++p) load(held[p], first + p);
#pragma unroll
        for (int p = 0; p < kI8ClHeld; ++p)
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) m[t] = M::join(m[t], held[p][t][i]);
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const uint32_t most = __reduce_max_sync(0xffffffffu, max(M::lo(m[t]), M::hi(m[t])));
        if (lane == 0) sh.most[wk * 4 + t] = most;
      }
      __syncwarp();
      cluster_sync();
      uint32_t most[4];
#pragma unroll
      for (int t = 0; t < 4; ++t)
        most[t] = lane < active ? peer_u32(cluster_addr(&sh.most[wk * 4 + t], (uint32_t)lane)) : 0u;
      TokenScale ts[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        most[t] = __reduce_max_sync(0xffffffffu, most[t]);
        ts[t] = token_scale(most[t]);
        if (lane == 0) sh.scale[wk * 4 + t] = ts[t].scale;
      }
      for (int first = 0; first < pieces; first += kI8ClHeld) {
        if (pieces > kI8ClHeld) {
#pragma unroll
          for (int p = 0; p < kI8ClHeld; ++p) load(held[p], first + p);
        }
#pragma unroll
        for (int p = 0; p < kI8ClHeld; ++p) {
          const int c = k0 + (first + p) * kI8ClPiece + lane * 8;
          if (c >= kq) break;
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const uint32_t keep = most[t] >= 0x7f800000u ? 0u : 0xffffffffu;
            uint32_t b[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float2 f = scaled2(M::value(held[p][t][2 * i]), ts[t].inverse, ts[t].inverse),
                           g = scaled2(M::value(held[p][t][2 * i + 1]), ts[t].inverse, ts[t].inverse);
              b[i] = low_bytes(f.x, f.y, g.x, g.y) & keep;
            }
            *reinterpret_cast<uint2*>(slot(wk * 4 + t, c) + (c & 8)) = make_uint2(b[0], b[1]);
          }
        }
      }
      __syncwarp();
    }
    fence_async_smem();
    mbar_arrive(&sh.quantised);
    // the partial sums take the place of the weights, which the products have read
    if (nkb > 0 && __all_sync(0xffffffffu, wait_or_abort(&sh.sums, 0, abort))) {
      tc_fence_after();
      const int q4 = warp & 3;
      const int m = wk >> 2;  // a warpgroup per tile of channels
      if (m < mt) {
        uint32_t r[32];
        tmem_ld32(tmem + (uint32_t)(m * kI8ClTokens) + ((uint32_t)(q4 * 32) << 16), r);
        tmem_ld_wait();
        if constexpr (W > 0) {  // [channel][token]
          int* at = part + (m * kI8BM + q4 * 32 + lane) * kI8ClRow;
#pragma unroll
          for (int i = 0; i < 8; ++i)
            *reinterpret_cast<uint4*>(at + 4 * i) = make_uint4(r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]);
        } else {  // [tile][token][channel]
          int* at = part + m * (kI8ClTokens * kI8ClCol) + q4 * 32 + lane;
#pragma unroll
          for (int i = 0; i < 32; ++i) at[i * kI8ClCol] = (int)r[i];
        }
      }
      tc_fence_before();
    }
    __syncwarp();
  }
  // Eight outputs along y's rows per worker: 1 / S of the cluster's.
  const int rows = mt * kI8BM / S, per = W > 0 ? kI8ClTokens / 8 : rows / 8;
  const int hi = ((int)threadIdx.x - 64) / per, lo = ((int)threadIdx.x - 64) - hi * per;
  const int row = rank * rows + (W > 0 ? hi : lo * 8), token = W > 0 ? lo * 8 : hi;  // of the cluster's
  const int n = n0 + row, v = v0 + token;
  const bool mine = warp >= 2 && (W > 0 ? hi < rows : hi < kI8ClTokens) && n < a.N && v < a.tokens;
  constexpr int kChans = W > 0 ? 1 : 8;
  float ws[kChans], bias[kChans];
#pragma unroll
  for (int e = 0; e < kChans; ++e) {
    ws[e] = mine && n + e < a.N ? a.ws[n + e] : 0.f;
    bias[e] = mine && n + e < a.N && a.bias != nullptr ? a.bias[n + e] : 0.f;
  }
  __syncwarp();
  cluster_sync();  // every CTA's partial sums
  if (mine) {
    constexpr int E = 16 / (int)sizeof(T);
    const int* at = part + (W > 0 ? row * kI8ClRow + token
                                  : row / kI8BM * (kI8ClTokens * kI8ClCol) + token * kI8ClCol + row % kI8BM);
    int4 r[8][2];
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      r[s][0] = r[s][1] = make_int4(0, 0, 0, 0);
      if (s >= active) continue;
      const uint32_t peer = cluster_addr(at, (uint32_t)s);
      r[s][0] = peer_int4(peer);
      r[s][1] = peer_int4(peer + 16);
    }
    int sum[8] = {};
#pragma unroll
    for (int s = 0; s < 8; ++s)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        sum[4 * h] += r[s][h].x;
        sum[4 * h + 1] += r[s][h].y;
        sum[4 * h + 2] += r[s][h].z;
        sum[4 * h + 3] += r[s][h].w;
      }
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int c = W > 0 ? 0 : e;
      f[e] = fmaf((float)sum[e] * sh.scale[W > 0 ? token + e : token], ws[c], bias[c]);
    }
    const int left = W > 0 ? a.tokens - v : a.N - n;  // of y's row
    T* out = static_cast<T*>(a.y) + (W > 0 ? ((long long)o * a.N + n) * a.inner + v : (long long)v * a.N + n);
#pragma unroll
    for (int h = 0; h < 8 / E; ++h) {
      if (a.vec_y) {  // y's rows are whole vectors
        if (h * E < left) *reinterpret_cast<uint4*>(out + h * E) = pack16<T>(f + h * E);
      } else {
#pragma unroll
        for (int e = h * E; e < (h + 1) * E; ++e)
          if (e < left) out[e] = from_acc<T>(f[e]);
      }
    }
  }
  __syncwarp();
  if (*abort && lane == 0) {
    if (warp == 0) drain_ring(sh.full, a.stages, issued);
    if (warp == 1) drain_mma(&sh.drain);
  }
  __syncwarp();
  cluster_sync();  // no CTA's memory is in use by the others any more
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, tmem_cols);
  }
}

// Whether the clusters take a product, and how: where K is long and all of them are resident at
// once (the occupancy query gives 15 clusters of 8, 33 of 4).  Tokens x K -> N in bf16, us,
// against the two kernels: channels first 512 x 2048 -> 512 13.9, 15.3; 512 x 1024 -> 256
// 9.0, 10.0; 64 x 2048 -> 512 8.7, 14.6; rows 16 x 4096 -> 1024 10.1, 18.4, 64 x 4096 -> 1024 13.7, 18.6.
// In two waves 216 x 2048 -> 2048 took 17.9, 15.4, and with a shorter K, rows 16 x 1024 -> 4096 9.0,
// 8.2, channels first 64 x 512 -> 512 7.4, 7.2 (rows are quantised faster).
bool cluster_takes(long long outer, int K, long long inner, int N, I8ClusterArgs* a) {
  const long long tokens = inner > 1 ? inner : outer, samples = inner > 1 ? outer : 1;
  const int kblocks = (K + kI8BK - 1) / kI8BK, mtiles = (N + kI8BM - 1) / kI8BM;
  if (kblocks < (inner > 1 ? 7 : 16) || tokens > 4096 || samples > 128) return false;
  a->tiles = (int)((tokens + kI8ClTokens - 1) / kI8ClTokens);
  const auto fits = [&](int S, int mt, int ctas) {
    a->S = S;
    a->mt = mt;
    a->slice = (kblocks + S - 1) / S;
    a->groups = (mtiles + mt - 1) / mt;
    return a->slice <= kI8ClSlice && samples * a->tiles * a->groups * S <= ctas;
  };
  return (kblocks >= 16 && fits(8, 1, 112)) || fits(4, 1, 128) || (kblocks >= 16 && mtiles > 1 && fits(4, 2, 128));
}

template <typename T>
int launch_cluster(I8ClusterArgs a, const int8_t* w, long long w_pitch, long long outer, cudaStream_t s) {
  a.tokens = a.inner > 1 ? a.inner : (int)outer;
  const bool chan = a.inner > 1, pair = sizeof(T) == 2 && a.inner % 2 == 0 && (reinterpret_cast<uintptr_t>(a.x) & 3) == 0;
  constexpr int E = 16 / (int)sizeof(T);
  a.vec_x = a.K % E == 0 && (reinterpret_cast<uintptr_t>(a.x) & 15) == 0;
  a.vec_y = (chan ? a.inner : a.N) % E == 0 && (reinterpret_cast<uintptr_t>(a.y) & 15) == 0;
  a.stages = std::min(kI8ClStages, a.mt * a.slice);
  const int sums = a.mt * (chan ? kI8BM * kI8ClRow : kI8ClTokens * kI8ClCol) * (int)sizeof(int);
  a.region = (std::max(a.stages * kI8BM * kI8BK, sums) + 1023) / 1024 * 1024;
  const size_t smem = (size_t)a.region + (size_t)a.slice * (kI8ClTokens * kI8BK) + 1024;
  CUtensorMap mW;
  if (!tma::encode_rows_8bit(&mW, w, a.K, a.N, 1, w_pitch, kI8BM)) {
    note_cuda_error(cudaErrorInvalidValue);
    return MEDNEXT_ERR_CUDA;
  }
  const auto run = [&](auto kern) {
    const int st = ensure_smem(kern, smem);
    if (st != MEDNEXT_OK) return st;
    const long long samples = chan ? outer : 1;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)a.S;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(samples * a.tiles * a.groups * a.S));
    cfg.blockDim = dim3(kI8Threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, kern, mW, a);
    return record_launch();
  };
  if (!chan) return run(i8_cluster_kernel<T, 0>);
  if constexpr (sizeof(T) == 2)
    if (pair) return run(i8_cluster_kernel<T, 2>);
  return run(i8_cluster_kernel<T, 1>);
}

int num_sms() {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0)
    return 148;
  return sms;
}

// Tensor maps of a product's operands (the tokens' with a matrix per sample) and, staged, of y.
template <typename T>
bool i8_maps(const I8GemmArgs& p, bool tokens_a, bool staged, const int8_t* a, long long a_pitch, const int8_t* b,
             long long b_pitch, uint32_t b_box, CUtensorMap* mA, CUtensorMap* mB, CUtensorMap* mY) {
  memset(mY, 0, sizeof(*mY));
  return tma::encode_rows_8bit(mA, a, p.K, p.a_rows, tokens_a ? p.samples : 1, a_pitch, kI8BM) &&
         tma::encode_rows_8bit(mB, b, p.K, p.b_rows, tokens_a ? 1 : p.samples, b_pitch, b_box) &&
         (!staged || tma::encode3<T>(mY, p.y, p.b_rows, p.a_rows, p.samples, 128 / sizeof(T), 32,
                                     CU_TENSOR_MAP_SWIZZLE_128B));
}

// ------------------------------ medium K in one kernel, channels first ------------------------------
// Between the narrow form and the large one (K up to 256, N up to 512), the 8-bit rows' way through
// memory is a third or more of the bytes, and two kernels are two ramps.  Here persistent CTAs keep
// the weights in shared memory (operand A) and take 256 bytes of each channel per tile (128 tokens
// of 16-bit data, 64 of fp32): one warp per 32 channels loads them into registers and quantises them into
// operand B; the product (tcgen05 kind::i8) goes into one of one to four accumulators, and other warps
// scale it and store it by TMA.
//
// The rows' length is what counts: read in 128-byte pieces of 256 channels, HBM gives 4.6 TB/s here,
// in 256-byte pieces 6.3.  (With 128-byte pieces, by TMA or by 16-byte asynchronous copies into a ring,
// 128 -> 32 channels at 64^3 took 33 us.)  A lane holds W neighbouring tokens; token W l + j is operand
// B's row 32 j + l, so that eight lanes' 16-byte stores meet different banks, and the accumulator's
// columns 32 j + l come together again in the registers of the thread that stores them.
//
// bf16, 64^3 voxels, against the two kernels: 128 -> 32 28.7 us, 42.5; 192 -> 64 40, 63; 128 -> 128 36, 48;
// 128 -> 512 93, 113; at 128^3 128 -> 32 150, 298 (4.5 TB/s); at 24^3 192 -> 64 7.9, 9.9.  What bounds it now is the
// turn of a group of quantising warps (its loads' latency and about 700 instructions).
constexpr int kI8MidK = 256;
constexpr int kI8MidWarps = 12, kI8MidGroups = 4;  // at most
constexpr int kI8MidScales = kI8MidGroups + kI8MaxAcc;

struct I8MidShared {
  uint64_t qfull[kI8MidGroups], qempty[kI8MidGroups];  // operand B
  uint64_t tfull[kI8MaxAcc], tempty[kI8MaxAcc];
  uint64_t weights, drain;
  uint32_t tmem_base;
  int abort;
  // Scales of the last tiles' tokens.  A tile's are written once the last product of its operand B is
  // done, which began after its accumulator's last tile was stored: as many as both have are enough.
  alignas(16) float scale[kI8MidScales][128];
  alignas(16) uint2 most[2][kI8MidWarps][32];  // by a warp's channels
};

// Whether one of the warps' threads failed: the same answer for all of a barrier's n threads.
__device__ __forceinline__ bool any_at_barrier(int id, int n, bool failed) {
  int any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.s32 p, %3, 0;\n\t"
      "barrier.cta.red.or.pred q, %1, %2, p;\n\t"
      "selp.s32 %0, 1, 0, q;\n\t}"
      : "=r"(any)
      : "r"(id), "r"(n), "r"((int)failed)
      : "memory");
  return any != 0;
}

// p: a_* the output channels, b_* the tokens; a_tiles and b_tiles count tiles of 128 channels and of
// bn tokens.  WARPS quantise, EPI scale and store.
template <typename T, int WARPS, int EPI>
__global__ void __launch_bounds__(32 * (2 + EPI + WARPS), 1)
    i8_mid_kernel(const T* __restrict__ x_all, const __grid_constant__ CUtensorMap mW,
                  const __grid_constant__ CUtensorMap mY, const __grid_constant__ I8GemmArgs p) {
  constexpr int W = 8 / (int)sizeof(T), TOK = 32 * W;  // tokens of a lane, of a tile
  extern __shared__ uint8_t i8_raw[];
  __shared__ I8MidShared sh;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kblocks = (p.K + kI8BK - 1) / kI8BK, mt = p.a_tiles, S = (p.K + 31) / 32;
  const int groups = p.groups, buffers = max(2, groups);  // of quantising warps, tiles in turn; of operand B
  const int q_bytes = kblocks * TOK * kI8BK;
  uint8_t* wsm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(i8_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* qsm = wsm + mt * kblocks * (kI8BM * kI8BK);
  uint8_t* stage = qsm + buffers * q_bytes;
  uint32_t tmem_cols = 32;
  while (tmem_cols < (uint32_t)(p.accs * mt * TOK)) tmem_cols *= 2;

  if (warp == 1) {
    tmem_alloc(&sh.tmem_base, tmem_cols);
    tmem_relinquish();
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < buffers; ++i) {
      mbar_init(&sh.qfull[i], 32 * S);
      mbar_init(&sh.qempty[i], 1);
    }
    for (int i = 0; i < p.accs; ++i) {
      mbar_init(&sh.tfull[i], 1);
      mbar_init(&sh.tempty[i], 32 * EPI);
    }
    mbar_init(&sh.weights, 1);
    mbar_init(&sh.drain, 1);
    sh.abort = 0;
    fence_mbarrier_init();
    tma_prefetch_map(&mW);
    tma_prefetch_map(&mY);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem_base;
  volatile int* abort = &sh.abort;
  const int tiles = p.b_tiles * p.samples;
  const int mine = (tiles - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x;
  const auto decode = [&](int i, int& sample, int& v0) {
    const int t = (int)blockIdx.x + i * (int)gridDim.x;
    sample = t / p.b_tiles;
    v0 = (t - sample * p.b_tiles) * TOK;
  };

  if (warp == 0) {
    if (lane == 0) {
      mbar_arrive_expect_tx(&sh.weights, (uint32_t)(mt * kblocks * (kI8BM * kI8BK)));
      for (int kb = 0; kb < kblocks; ++kb)
        for (int m = 0; m < mt; ++m)
          for (int r = 0; r < p.copies; ++r)
            tma_load_3d(wsm + (kb * mt + m) * (kI8BM * kI8BK) + r * (kI8BM / p.copies * kI8BK), &mW, &sh.weights, kb * kI8BK,
                        m * kI8BM, 0);
    }
  } else if (warp == 1) {
    if (lane == 0 && wait_or_abort(&sh.weights, 0, abort)) {
      const uint32_t idesc = make_idesc_i8(kI8BM, TOK);
      RingAt q, acc;
      for (int i = 0; i < mine; ++i, q.next(buffers), acc.next(p.accs)) {
        if (acc.turn > 0 && !wait_or_abort(&sh.tempty[acc.slot], (acc.turn - 1) & 1, abort)) break;
        if (!wait_or_abort(&sh.qfull[q.slot], q.turn & 1, abort)) break;
        tc_fence_after();
        const uint32_t d = tmem + (uint32_t)(acc.slot * mt * TOK);
        for (int kb = 0; kb < kblocks; ++kb) {
          const uint32_t sb = smem_u32(qsm + q.slot * q_bytes + kb * (TOK * kI8BK));
          const int steps = min(kI8BK, p.K - kb * kI8BK + 31) / 32;  // zeros past K
          for (int m = 0; m < mt; ++m) {
            const uint32_t sa = smem_u32(wsm + (kb * mt + m) * (kI8BM * kI8BK));
            for (int ks = 0; ks < steps; ++ks)
              mma_i8_ss(d + (uint32_t)(m * TOK), make_sw128_desc(sa + ks * 32, 16, 1024),
                        make_sw128_desc(sb + ks * 32, 16, 1024), idesc, kb > 0 || ks > 0 ? 1u : 0u);
          }
        }
        mma_commit(&sh.qempty[q.slot]);
        mma_commit(&sh.tfull[acc.slot]);
      }
    }
  } else if (warp < 2 + EPI) {
    // Pieces of 32 channels x 128 bytes of tokens, in turn among the groups of four warps.  A warp reads
    // 32 of the accumulator's 128 lanes: with 64 channels or fewer they are there twice, with 32 four
    // times, and the copies' warps take pieces in turn too.
    constexpr int E = 16 / (int)sizeof(T);
    const int e = warp - 2, q4 = warp & 3, q_chan = q4 % (4 / p.copies);
    const int sharers = EPI / 4 * p.copies, me = (e >> 2) * p.copies + q4 / (4 / p.copies);
    int turn = 0;  // of the next tile's first piece
    uint8_t* stg = stage + e * kI8StageBytes;
    RingAt acc;
    for (int i = 0; i < mine; ++i, acc.next(p.accs)) {
      int sample, v0;
      decode(i, sample, v0);
      if (!__all_sync(0xffffffffu, wait_or_abort(&sh.tfull[acc.slot], acc.turn & 1, abort))) break;
      tc_fence_after();
      const float* scales = sh.scale[i % kI8MidScales];
      for (int piece = 0; piece < 2 * mt; ++piece) {
        const bool my_turn = turn == me;
        if (++turn == sharers) turn = 0;
        const int m = piece >> 1, c = piece & 1, r0 = m * kI8BM + q_chan * 32, n = r0 + lane;
        if (!my_turn || r0 >= p.a_rows) continue;
        if (v0 + c * (16 * W) >= p.b_rows) continue;
        uint32_t r[W][16];
        const uint32_t at = tmem + (uint32_t)((acc.slot * mt + m) * TOK + 16 * c) + ((uint32_t)(q4 * 32) << 16);
#pragma unroll
        for (int j = 0; j < W; ++j) tmem_ld16(at + 32 * j, r[j]);
        const float ws = n < p.a_rows ? p.a_scale[n] : 0.f, bias = n < p.a_rows && p.bias != nullptr ? p.bias[n] : 0.f;
        if (lane == 0) bulk_wait_read<0>();  // the last store has read the buffer
        __syncwarp();
        tmem_ld_wait();
#pragma unroll
        for (int u = 0; u < 8; ++u) {  // 16 bytes of tokens
          float f[E];
#pragma unroll
          for (int h = 0; h < E; h += 4) {
            const float4 ts = *reinterpret_cast<const float4*>(scales + c * (16 * W) + u * E + h);
            const float tv[4] = {ts.x, ts.y, ts.z, ts.w};
#pragma unroll
            for (int k = 0; k < 4; k += 2) {
              const int t = u * E + h + k;  // token of the piece: W i + j
              const float2 v = make_float2((float)(int)r[t % W][t / W], (float)(int)r[(t + 1) % W][(t + 1) / W]);
              const float2 o = __ffma2_rn(__fmul2_rn(v, make_float2(tv[k], tv[k + 1])), make_float2(ws, ws),
                                          make_float2(bias, bias));
              f[h + k] = o.x;
              f[h + k + 1] = o.y;
            }
          }
          *reinterpret_cast<uint4*>(stg + lane * 128 + ((u ^ (lane & 7)) << 4)) = pack16<T>(f);
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) {
          tma_store_3d(&mY, stg, v0 + c * (16 * W), r0, sample);
          bulk_commit();
        }
      }
      __syncwarp();
      tc_fence_before();
      mbar_arrive(&sh.tempty[acc.slot]);
    }
    if (lane == 0) bulk_wait_all();
  } else {
    const int u = warp - 2 - EPI, group = u / S, s = u - group * S;
    if (group < groups) {
      const int rows = min(32, p.K - s * 32);  // channels of this warp
      uint32_t xa[32], xb[32];
      const auto load = [&](int i) {
        int sample, v0;
        decode(i, sample, v0);
        const int v = v0 + lane * W;
        const bool in = i < mine && v < p.b_rows;  // b_rows is a multiple of W
        const T* px = x_all + ((long long)sample * p.K + s * 32) * p.b_rows + v;
#pragma unroll
        for (int k = 0; k < 32; ++k) {
          const uint2 w = in && k < rows ? *reinterpret_cast<const uint2*>(px) : make_uint2(0u, 0u);
          xa[k] = w.x;
          xb[k] = w.y;
          px += p.b_rows;
          asm volatile("" : "+l"(px));  // one address in flight, not 32
        }
      };
      load(group);
      bool failed = false;
      for (int i = group, turn = 0; i < mine; i += groups, ++turn) {
        uint2 m = make_uint2(0u, 0u);
        const auto join = [](uint32_t a, uint32_t b) { return sizeof(T) == 2 ? __vmaxu2(a, b) : max(a, b); };
        constexpr uint32_t kMag = sizeof(T) == 2 ? 0x7fff7fffu : 0x7fffffffu;
#pragma unroll
        for (int k = 0; k < 32; ++k) m = make_uint2(join(m.x, xa[k] & kMag), join(m.y, xb[k] & kMag));
        uint2(*maxima)[32] = sh.most[turn & 1] + group * S;
        maxima[s][lane] = m;
        // a warp that gave up says so here: the group leaves together
        if (any_at_barrier(1 + group, 32 * S, failed)) break;
        for (int r = 0; r < S; ++r) {
          const uint2 other = maxima[r][lane];
          m = make_uint2(join(m.x, other.x), join(m.y, other.y));
        }
        uint32_t most[W];
        if constexpr (sizeof(T) == 2) {
          most[0] = Mag<T>::lo(m.x);
          most[1] = Mag<T>::hi(m.x);
          most[2] = Mag<T>::lo(m.y);
          most[3] = Mag<T>::hi(m.y);
        } else {
          most[0] = m.x;
          most[1] = m.y;
        }
        TokenScale ts[W];
#pragma unroll
        for (int j = 0; j < W; ++j) ts[j].inverse = token_inverse(most[j]);
        // this operand B's last product is done
        const int q = groups > 1 ? group : turn & 1, use = groups > 1 ? turn : turn >> 1;
        failed = use > 0 && !__all_sync(0xffffffffu, wait_or_abort(&sh.qempty[q], (uint32_t)((use - 1) & 1), abort));
        if (failed) continue;
        if (s == 0) {
#pragma unroll
          for (int j = 0; j < W; ++j) sh.scale[i % kI8MidScales][lane * W + j] = token_scale(most[j]).scale;
        }
        uint8_t* dst = qsm + q * q_bytes + (s >> 2) * (TOK * kI8BK) + lane * kI8BK;
        constexpr int WH = W / 2;  // tokens of a word
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const TokenScale(&th)[WH] = *reinterpret_cast<const TokenScale(*)[WH]>(ts + half * WH);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t b[WH][4];
            quantize16<T, WH>((half == 0 ? xa : xb) + h * 16, th, b);
#pragma unroll
            for (int j = 0; j < WH; ++j) {
              const uint32_t keep = most[half * WH + j] >= 0x7f800000u ? 0u : 0xffffffffu;
              *reinterpret_cast<uint4*>(dst + (half * WH + j) * (32 * kI8BK) + ((((s & 3) * 2 + h) ^ (lane & 7)) << 4)) =
                  make_uint4(b[j][0] & keep, b[j][1] & keep, b[j][2] & keep, b[j][3] & keep);
            }
          }
        }
        fence_async_smem();
        mbar_arrive(&sh.qfull[q]);
        load(i + groups);
      }
    }
  }
  __syncthreads();
  if (*abort && lane == 0) {
    if (warp == 0) mbar_wait(&sh.weights, 0);
    if (warp == 1) drain_mma(&sh.drain);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, tmem_cols);
  }
}

// Groups of quantising warps (one warp per 32 channels): as many as there is room for.  False: not even one.
bool mid_plan(int K, int N, int tok, int warps, int epi, int* groups, size_t* smem) {
  const size_t kblocks = (K + kI8BK - 1) / kI8BK, mt = (N + kI8BM - 1) / kI8BM;
  for (int g = std::min(kI8MidGroups, warps / ((K + 31) / 32)); g >= 1; --g) {
    *groups = g;
    *smem = kblocks * (mt * kI8BM + std::max(2, g) * tok) * kI8BK + (size_t)epi * kI8StageBytes + 1024;
    if (*smem <= 227 * 1024 - sizeof(I8MidShared)) return true;
  }
  return false;
}
// Whether the medium form takes a product: whole 16-byte rows of y, room, and tiles enough for the SMs (108
// tiles: 192 -> 64 7.9 us, two kernels 9.9, but 96 -> 32 9.0, 8.5).
bool mid_takes(const void* x, const void* y, long long outer, int K, long long inner, int N, size_t esz) {
  const int tok = 256 / (int)esz;
  const long long tiles = outer * ((inner + tok - 1) / tok);
  int groups;
  size_t smem;
  return K <= kI8MidK && N <= 4 * kI8BM && inner % (16 / (long long)esz) == 0 && reinterpret_cast<uintptr_t>(x) % 8 == 0 &&
         reinterpret_cast<uintptr_t>(y) % 16 == 0 && mid_plan(K, N, tok, 8, 8, &groups, &smem) &&
         tiles >= (K > 96 ? 64 : kI8Sms) && tiles < ((long long)1 << 30);
}

template <typename T>
int launch_mid(const void* x, const int8_t* w, const float* ws, long long w_pitch, const float* bias, void* y,
               long long outer, int K, long long inner, int N, cudaStream_t s) {
  constexpr int tok = 256 / (int)sizeof(T);
  I8GemmArgs p{};
  p.a_scale = ws;
  p.bias = bias;
  p.y = y;
  p.a_rows = N;
  p.b_rows = (int)inner;
  p.K = K;
  p.N = N;
  p.bn = tok;
  p.a_tiles = (N + kI8BM - 1) / kI8BM;
  p.b_tiles = (int)((inner + tok - 1) / tok);
  p.samples = (int)outer;
  p.accs = std::min(kI8MaxAcc, 512 / (p.a_tiles * tok));
  p.copies = N <= 32 ? 4 : (N <= 64 ? 2 : 1);
  CUtensorMap mW, mY;
  if (!tma::encode_rows_8bit(&mW, w, K, N, 1, w_pitch, kI8BM / p.copies) ||
      !tma::encode3<T>(&mY, y, inner, N, outer, tok / 2, 32, CU_TENSOR_MAP_SWIZZLE_128B)) {
    note_cuda_error(cudaErrorInvalidValue);
    return MEDNEXT_ERR_CUDA;
  }
  const auto run = [&](auto kern, int warps, int epi) {
    size_t smem;
    if (!mid_plan(K, N, tok, warps, epi, &p.groups, &smem)) return (int)MEDNEXT_ERR_BAD_SHAPE;
    const int st = ensure_smem(kern, smem);
    if (st != MEDNEXT_OK) return st;
    const long long tiles = (long long)p.b_tiles * outer;
    kern<<<(unsigned)std::min<long long>(tiles, num_sms()), 32 * (2 + epi + warps), smem, s>>>(static_cast<const T*>(x), mW, mY,
                                                                                               p);
    return record_launch();
  };
  // few outputs leave the work to the quantising warps (64^3, bf16: 192 -> 64 40 us, with 10 and 8 warps 52),
  // many to the storing ones (128 -> 512 94 us, with 12 and 4 warps 117)
  return N <= 64 ? run(i8_mid_kernel<T, 12, 4>, 12, 4) : run(i8_mid_kernel<T, 10, 8>, 10, 8);
}

// q: [outer * inner][q_pitch], w: [N][w_pitch]; y [outer, N, inner]
template <typename T>
int launch_gemm(const int8_t* q, const float* qs, long long q_pitch, const int8_t* w, const float* ws,
                long long w_pitch, const float* bias, void* y, long long outer, long long inner, int K, int N,
                cudaStream_t s) {
  const bool chan = inner > 1;
  const long long tokens = chan ? inner : outer;  // of a sample
  const bool staged = (chan ? inner : N) % (16 / (long long)sizeof(T)) == 0 && reinterpret_cast<uintptr_t>(y) % 16 == 0;
  const bool tokens_a = staged != chan;
  const int8_t *a = tokens_a ? q : w, *b = tokens_a ? w : q;
  const long long a_pitch = tokens_a ? q_pitch : w_pitch, b_pitch = tokens_a ? w_pitch : q_pitch;
  I8GemmArgs p{};
  p.a_scale = tokens_a ? qs : ws;
  p.b_scale = tokens_a ? ws : qs;
  p.bias = bias;
  p.y = y;
  p.a_rows = tokens_a ? (int)tokens : N;
  p.b_rows = tokens_a ? N : (int)tokens;
  p.samples = chan ? (int)outer : 1;
  p.K = K;
  p.N = N;
  const int sms = num_sms();
  CUtensorMap mA, mB, mY;
  const auto no_map = [] {
    note_cuda_error(cudaErrorInvalidValue);
    return (int)MEDNEXT_ERR_CUDA;
  };
  const auto run = [&](auto kern, unsigned grid, size_t smem) {
    const int st = ensure_smem(kern, smem);
    if (st != MEDNEXT_OK) return st;
    return launch_dependent(kern, dim3(grid), dim3(kI8Threads), smem, s, mA, mB, mY, p);
  };
  const int staging = staged ? kI8EpiWarps * kI8StageBytes : 0;

  // Pairs of SMs where both halves of the tiles are mostly full and every pair has one
  // (32768 x 1024 -> 4096 bf16, the product alone: 118 us against 149).
  const long long pair_tiles = (long long)((p.a_rows + 255) / 256) * ((p.b_rows + 255) / 256) * p.samples;
  if (staged && K >= 256 && p.a_rows > 128 && p.b_rows > 128 && pair_tiles >= sms / 2) {
    if (pair_tiles >= ((long long)1 << 31)) return MEDNEXT_ERR_BAD_SHAPE;
    p.bn = 256;
    p.a_tiles = (p.a_rows + 255) / 256;
    p.b_tiles = (p.b_rows + 255) / 256;
    if (!i8_maps<T>(p, tokens_a, staged, a, a_pitch, b, b_pitch, kI8BM, &mA, &mB, &mY)) return no_map();
    const size_t smem = (size_t)kI8PairStages * 2 * kI8BM * kI8BK + staging + 1024;
    const unsigned grid = 2 * (unsigned)std::min<long long>(pair_tiles, sms / 2);
    return tokens_a ? run(i8_gemm_pair_kernel<T, true>, grid, smem) : run(i8_gemm_pair_kernel<T, false>, grid, smem);
  }

  p.a_tiles = (p.a_rows + kI8BM - 1) / kI8BM;
  const long long a_all = (long long)p.a_tiles * p.samples;
  // the widest B tile that still gives every SM a tile, at most what B fills; at least a
  // staged store's columns
  const int least = staged ? std::max(32, 128 / (int)sizeof(T)) : 32;
  p.bn = 256;
  while (p.bn > least && (p.bn / 2 >= p.b_rows || a_all * ((p.b_rows + p.bn - 1) / p.bn) < sms)) p.bn /= 2;
  p.b_tiles = (p.b_rows + p.bn - 1) / p.bn;
  const long long tiles = a_all * p.b_tiles;
  if (tiles >= ((long long)1 << 31)) return MEDNEXT_ERR_BAD_SHAPE;
  p.accs = std::min(kI8MaxAcc, 512 / p.bn);
  p.share = p.accs < 4 || tiles <= sms;
  const int ring = kI8BM * kI8BK + p.bn * kI8BK;
  p.stages = std::min(kI8MaxStages, (216 * 1024 - staging) / ring);
  if (!i8_maps<T>(p, tokens_a, staged, a, a_pitch, b, b_pitch, p.bn, &mA, &mB, &mY)) return no_map();
  const size_t smem = (size_t)p.stages * ring + staging + 1024;
  const unsigned grid = (unsigned)std::min<long long>(tiles, sms);
  if (staged)
    return tokens_a ? run(i8_gemm_kernel<T, true, true>, grid, smem) : run(i8_gemm_kernel<T, false, true>, grid, smem);
  return tokens_a ? run(i8_gemm_kernel<T, true, false>, grid, smem) : run(i8_gemm_kernel<T, false, false>, grid, smem);
}

long long pitch16(int64_t k) { return (k + 15) / 16 * 16; }

template <typename T>
int launch_quantize(const void* xv, int8_t* q, float* scale, long long outer, int K, long long inner, long long pitch,
                    cudaStream_t s) {
  const long long tokens = outer * inner;
  const T* x = static_cast<const T*>(xv);
  if (inner > 1) {
    const bool pair = sizeof(T) == 2 && inner % 2 == 0 && (reinterpret_cast<uintptr_t>(xv) & 3) == 0;
    auto run = [&](auto kern, int W, int TX, int piece) {
      const int S = (int)std::min<long long>(32, (pitch + piece - 1) / piece), P = std::max(1, 4 / S);
      const long long tiles = outer * ((inner + TX * W - 1) / (TX * W));
      const unsigned grid = (unsigned)std::min<long long>((tiles + P - 1) / P, kI8Sms * 64);
      kern<<<grid, dim3(32, S, P), 2 * (size_t)P * S * W * TX * sizeof(uint32_t), s>>>(x, q, scale, (int)outer,
                                                                                       (int)inner, K, (int)pitch);
      return record_launch();
    };
    const bool few = outer * ((inner + 63) / 64) < kI8Sms;
    if constexpr (sizeof(T) == 2)
      if (pair) return few ? run(i8_quantize_chan_kernel<T, 2, 8, 16>, 2, 8, 64) : run(i8_quantize_chan_kernel<T, 2, 32, 32>, 2, 32, 32);
    return few ? run(i8_quantize_chan_kernel<T, 1, 8, 16>, 1, 8, 64) : run(i8_quantize_chan_kernel<T, 1, 32, 32>, 1, 32, 32);
  }
  constexpr int E = 16 / sizeof(T);
  const int vecs = (int)((pitch + E - 1) / E);
  // the registers of a warp hold 16 vectors per lane: 2048 columns of fp32, 4096 of 16 bits (wider ones go by
  // single elements: 8192 x 4096 fp32 58 us, bf16 here 21)
  if (K % E == 0 && (reinterpret_cast<uintptr_t>(xv) & 15) == 0 && pitch - K < 16 && vecs <= 512) {
    int G = 1;
    while (G < 32 && G < vecs) G *= 2;
    const int rows = 256 / G;
    const unsigned grid = (unsigned)std::min<long long>((tokens + rows - 1) / rows, kI8Sms * 64);
    if (vecs <= 32) i8_quantize_rows_kernel<T, 1><<<grid, 256, 0, s>>>(x, q, scale, tokens, K, (int)pitch, G);
    else if (vecs <= 128) i8_quantize_rows_kernel<T, 4><<<grid, 256, 0, s>>>(x, q, scale, tokens, K, (int)pitch, G);
    else i8_quantize_rows_kernel<T, 16><<<grid, 256, 0, s>>>(x, q, scale, tokens, K, (int)pitch, G);
    return record_launch();
  }
  const auto any = [&](auto steps) {
    constexpr int kSteps = decltype(steps)::value;
    if constexpr (sizeof(T) == 2 && kSteps >= 4)
      if (K <= 2048 && tokens >= kI8Sms * 64LL) {  // several blocks for each resident CTA
        const size_t smem = 2 * (size_t)block_bytes<T>(8, K);
        const int st = ensure_smem(i8_quantize_any_kernel<T, true, kSteps>, smem);
        if (st != MEDNEXT_OK) return st;
        i8_quantize_any_kernel<T, true, kSteps><<<kI8Sms * (kSteps < 8 ? 4 : 2), 256, smem, s>>>(x, q, scale, tokens, K,
                                                                                                 (int)pitch);
        return record_launch();
      }
    i8_quantize_any_kernel<T, false, kSteps><<<(unsigned)std::min<long long>((tokens + 7) / 8, kI8Sms * 16), 256, 0, s>>>(
        x, q, scale, tokens, K, (int)pitch);
    return record_launch();
  };
  if (pitch <= 128) return any(std::integral_constant<int, 1>{});
  if (pitch <= 256) return any(std::integral_constant<int, 2>{});
  if (pitch <= 512) return any(std::integral_constant<int, 4>{});
  return any(std::integral_constant<int, 8>{});
}

template <typename T>
int launch_narrow(I8NarrowArgs a, cudaStream_t s) {
  constexpr int W = kNarrowW<T>;
  const int S = (a.K + 31) / 32, P = 4 / S;
  const size_t smem = narrow_smem(a.K, a.N, W, P);
  narrow_share(a.N, S, &a.mt_warp, &a.mt_store);
  const long long tiles = (long long)a.outer * ((a.inner + 32 * W - 1) / (32 * W));
  // four turns of the resident CTAs, so that SMs that are done early take more
  const int per_sm = std::max(1, std::min(kNarrowWarps / (S * P), (int)(227 * 1024 / (smem + 1024))));
  const unsigned grid = (unsigned)std::min((tiles + P - 1) / P, 4LL * kI8Sms * per_sm);
  CUtensorMap mY;
  if (!tma::encode3<T>(&mY, a.y, a.inner, a.N, a.outer, 32 * W, 16 * a.mt_store, CU_TENSOR_MAP_SWIZZLE_128B)) {
    note_cuda_error(cudaErrorInvalidValue);
    return MEDNEXT_ERR_CUDA;
  }
  auto run = [&](auto kern) {
    const int st = ensure_smem(kern, smem);
    if (st != MEDNEXT_OK) return st;
    kern<<<grid, dim3(32, S, P), smem, s>>>(mY, a);
    return record_launch();
  };
  return S == 1 ? run(i8_narrow_kernel<T, 1>) : run(i8_narrow_kernel<T, 2>);
}

template <typename T>
int launch_linear(const void* x, const int8_t* w, const float* ws, long long w_pitch, const float* bias, void* y,
                  int8_t* q, float* qs, long long outer, int K, long long inner, int N, cudaStream_t s) {
  if (few_takes(outer * inner, K)) {
    I8FewArgs a{};
    a.x = x; a.w = w; a.ws = ws; a.bias = bias; a.y = y;
    a.w_pitch = w_pitch;
    a.tokens = (int)(outer * inner); a.inner = (int)inner; a.K = K; a.N = N;
    return launch_few<T>(a, s);
  }
  if (inner > 1 && narrow_takes(x, y, outer, K, inner, N, sizeof(T))) {
    I8NarrowArgs a{};
    a.x = x; a.w = w; a.ws = ws; a.bias = bias; a.y = y;
    a.w_pitch = w_pitch;
    a.outer = (int)outer; a.inner = (int)inner; a.K = K; a.N = N;
    return launch_narrow<T>(a, s);
  }
  I8ClusterArgs c{};
  if (cluster_takes(outer, K, inner, N, &c)) {
    c.x = x; c.ws = ws; c.bias = bias; c.y = y;
    c.inner = (int)inner; c.K = K; c.N = N;
    return launch_cluster<T>(c, w, w_pitch, outer, s);
  }
  if (inner > 1 && mid_takes(x, y, outer, K, inner, N, sizeof(T)))
    return launch_mid<T>(x, w, ws, w_pitch, bias, y, outer, K, inner, N, s);
  int st = launch_quantize<T>(x, q, qs, outer, K, inner, pitch16(K), s);
  if (st != MEDNEXT_OK) return st;
  return launch_gemm<T>(q, qs, pitch16(K), w, ws, w_pitch, bias, y, outer, inner, K, N, s);
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

// The workspace holds the tokens' 8-bit rows, then their scales; the forms that quantise into
// shared memory for any alignment need none.
size_t mednext_int8_linear_workspace_size(int64_t outer, int64_t k, int64_t inner, int64_t n, int dtype) {
  if (i8_check(outer, k, inner, dtype) != MEDNEXT_OK || n <= 0 || n > kI8MaxN) return 0;
  I8ClusterArgs c{};
  if (few_takes(outer * inner, (int)k) || cluster_takes(outer, (int)k, inner, (int)n, &c)) return 0;
  const size_t tokens = (size_t)(outer * inner);
  return tokens * (size_t)pitch16(k) + (tokens * sizeof(float) + 15) / 16 * 16;
}

int mednext_int8_linear(const void* x, const int8_t* weight, const float* weight_scale, const float* bias, void* y,
                        void* workspace, size_t workspace_bytes, int64_t outer, int64_t k, int64_t inner, int64_t n,
                        int64_t weight_pitch, int dtype, mednext_stream_t stream) {
  const int st = i8_check(outer, k, inner, dtype);
  if (st != MEDNEXT_OK) return st;
  if (n <= 0 || n > kI8MaxN || weight_pitch < k || weight_pitch % 16 != 0 ||
      weight_pitch > ((int64_t)1 << 30))
    return MEDNEXT_ERR_BAD_SHAPE;
  if (outer * inner == 0) return MEDNEXT_OK;
  if (x == nullptr || weight == nullptr || weight_scale == nullptr || y == nullptr) return MEDNEXT_ERR_NULL_POINTER;
  if (off(x, elem_size(dtype)) || off(y, elem_size(dtype)) || off(weight, 16) || off(weight_scale, 4) || off(bias, 4))
    return MEDNEXT_ERR_ALIGNMENT;
  const size_t need = mednext_int8_linear_workspace_size(outer, k, inner, n, dtype);
  if (need > 0 && (workspace == nullptr || off(workspace, 16) || workspace_bytes < need)) return MEDNEXT_ERR_WORKSPACE;
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
