// Low-rank adapters of many requests beside a shared projection:
//   out[t] = base[t] + s_a (x[t] . down_a^T) up_a,   a the adapter of token t,
// down (L, r, K) and up (L, r, N), both with the long side contiguous, so that
// three kernels do the forward and the backward pass:
//   shrink  h = x . down^T   and   u = g . up^T       (contraction over the long side)
//   expand  out = base + s h . up   and   gx = s u . down   (contraction over the rank)
//   outer   gdown = s u^T x   and   gup = s h^T g      (contraction over the tokens)
// on the 16x16x32 matrix instructions, with f32 sums.  All three are bound by
// reading and writing the token rows: at rank 64 they do 64 flops a byte, the
// card's balance is above 300.
//
// The contraction index of a matrix instruction is free as long as both
// operands agree on it, and so is the order of output columns.  Shrink gives a
// lane 16 consecutive elements of a row per pair of instructions (whole
// 128-byte lines a wave).  Expand and outer need operands whose contraction
// index runs across rows: a lane loads 16 bytes (8 columns) of 8 rows, and one
// byte permute per register pairs two rows of a column, which gives 8 operands
// for columns 8i + j (i the lane, j the operand) without going through LDS;
// the outputs of the 8 instructions are 8 consecutive columns of a lane.
//
// h and u enter the second products as two bf16 terms (16 bits of mantissa;
// f16 tensors: two f16 terms of a row scaled by a power of two, or the f16
// operand as two bf16 terms), so that only the outputs are rounded to the
// tensors' type.
#include <math.h>

#include "mxgg_device.h"
#include "mxgg_host.h"

namespace mxgg {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));

constexpr int kLoraThreads = 256;
constexpr int kLoraWaves = kLoraThreads / kWave;
constexpr int kMaxRank = 512;
constexpr int kMaxAdapters = 1024;
constexpr int kExpandRows = 64;      // tokens of an expand workgroup, 16 a wave
constexpr int kExpandCols = 128;     // and its columns at a time
constexpr int kPassRows = 64;        // tokens a workgroup looks over for those without an adapter
constexpr int kOuterCols = 128;      // columns of an outer workgroup

template <typename T>
struct Mat;
template <>
struct Mat<__bf16> {
  static __device__ __forceinline__ v4f mma(v4u a, v4u b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
  }
};
template <>
struct Mat<_Float16> {
  static __device__ __forceinline__ v4f mma(v4u a, v4u b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
  }
};

// 8 elements at p, `left` of them in range (zeros past them); any alignment.
template <typename T, bool ONCE = false>
__device__ __forceinline__ v4u load8(const T* p, int64_t left) {
  v4u r;
  if (left >= 8) {
    r = ONCE ? load_any_once(p) : load_any(p);
  } else {
    T v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < left ? p[i] : (T)0.f;
    __builtin_memcpy(&r, v, 16);
  }
  return r;
}

template <typename T, bool ONCE = false>
__device__ __forceinline__ void store8(T* p, const T (&v)[8], int64_t left) {
  if (left >= 8) {
    v4u r;
    __builtin_memcpy(&r, v, 16);
    if (ONCE) store_any_once(p, r);
    else store_any(p, r);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) p[i] = v[i];
  }
}

// Operand from 8 rows of 16-bit columns: column j of all rows.
template <typename V>
__device__ __forceinline__ v4u column_of(const V (&row)[8], int j) {
  const uint32_t sel = j & 1 ? 0x07060302u : 0x05040100u;
  v4u r;
#pragma unroll
  for (int p = 0; p < 4; ++p) r[p] = __builtin_amdgcn_perm(row[2 * p + 1][j >> 1], row[2 * p][j >> 1], sel);
  return r;
}

// x = hi + lo in two terms of T; the second term of an infinity or NaN is 0.
template <typename T>
__device__ __forceinline__ void two_terms(const float (&x)[8], v4u& hi, v4u& lo) {
  T h[8], l[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    h[i] = (T)x[i];
    const float rest = x[i] - (float)h[i];
    l[i] = (T)(fabsf(rest) < INFINITY ? rest : 0.f);
  }
  __builtin_memcpy(&hi, h, 16);
  __builtin_memcpy(&lo, l, 16);
}

// An f16 operand as two bf16 terms (exact: 11 bits in 16).
__device__ __forceinline__ void two_terms_f16(v4u x, v4u& hi, v4u& lo) {
  _Float16 h[8];
  float f[8];
  __builtin_memcpy(h, &x, 16);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = (float)h[i];
  two_terms<__bf16>(f, hi, lo);
}

// Power of two that brings a row with largest magnitude `top` (bits) into [1, 2)
// (down) or back; 1 for rows that are zero, not finite, or beyond 2^+-120.
__device__ __forceinline__ float row_scale(uint32_t top, bool down) {
  const uint32_t e = top & 0x7f800000u;
  if (e < (7u << 23) || e > (247u << 23)) return 1.f;
  return __uint_as_float(down ? 0x7f000000u - e : e);
}

// The largest magnitude (bits) of v and top.
__device__ __forceinline__ uint32_t top_bits(const float (&v)[8], uint32_t top) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t a = abs_bits(v[i]);
    top = a > top ? a : top;
  }
  return top;
}

// The `BM`-row tile t of the tokens sorted by adapter.
template <int BM>
__device__ __forceinline__ TileRoute lora_tile(const int32_t* __restrict__ offs, int L, int t) {
  int pn;
  return route_tile(offs, L, BM, 1, 1, t, pn);
}

// ---------------------------------------------------------------------------
// shrink: h[s][pos][rank] = sum over split s of x[src[pos]] . w[adapter][rank]
// ---------------------------------------------------------------------------

template <typename T, int MT, int NT>
struct ShrinkStep {
  v4u a[MT][2], b[NT][2];
};

// Workgroup: 16 MT tokens of one adapter, 16 NT ranks, 1/S of the long side,
// whose 64-element steps go round its four waves; their sums are joined in LDS,
// the splits' by the reader.  Rows are read once, the adapter once per tile.
template <typename T, int MT, int NT>
__global__ __launch_bounds__(kLoraThreads, MT * NT == 16 && NT == 8 ? 1 : 2) void lora_shrink_kernel(const T* __restrict__ x, int64_t ldx, int64_t K,
                                                                      const T* __restrict__ w, int64_t ldw_r,
                                                                      int64_t ldw_l, int r,
                                                                      const int32_t* __restrict__ src,
                                                                      const int32_t* __restrict__ offs, int L, int64_t M,
                                                                      float* __restrict__ h, int RP) {
  constexpr int BM = 16 * MT, BN = 16 * NT;
  __shared__ v4f red[2][MT * NT][kWave];
  const TileRoute tile = lora_tile<BM>(offs, L, blockIdx.x);
  if (tile.expert < 0) return;
  const int lane = threadIdx.x & (kWave - 1), n16 = lane & 15, q = lane >> 4, w4 = wave_id();
  const int64_t pos0 = tile.start + (int64_t)tile.block * BM;
  const int rank0 = blockIdx.z * BN;
  const T* xp[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int row = i * 16 + n16;
    const int t = row < tile.rows ? src[pos0 + row] : 0;
    xp[i] = x + (int64_t)(t > 0 ? t : 0) * ldx + q * 16;       // rows outside the tile give sums nobody stores
  }
  const T* wp[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const int rank = rank0 + i * 16 + n16;
    wp[i] = w + tile.expert * ldw_l + (int64_t)(rank < r ? rank : r - 1) * ldw_r + q * 16;
  }
  const int64_t steps = (K + 63) / 64, per = (steps + gridDim.y - 1) / gridDim.y;
  const int64_t s0 = blockIdx.y * per, s1 = s0 + per < steps ? s0 + per : steps;
  v4f acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};

  auto load = [&](ShrinkStep<T, MT, NT>& f, int64_t st) {
    const int64_t k = st * 64;
    if (k + 64 <= K) {
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int c = 0; c < 2; ++c) f.a[i][c] = load8(xp[i] + k + 8 * c, 8);
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int c = 0; c < 2; ++c) f.b[i][c] = load8(wp[i] + k + 8 * c, 8);
    } else {
      const int64_t left = K - k - q * 16;
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int c = 0; c < 2; ++c) f.a[i][c] = load8(xp[i] + k + 8 * c, left - 8 * c);
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int c = 0; c < 2; ++c) f.b[i][c] = load8(wp[i] + k + 8 * c, left - 8 * c);
    }
  };
  auto mma = [&](const ShrinkStep<T, MT, NT>& f) {
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = Mat<T>::mma(f.a[i][c], f.b[j][c], acc[i][j]);
  };
  ShrinkStep<T, MT, NT> f0, f1;
  int64_t st = s0 + w4;
  if (st < s1) load(f0, st);
  while (st < s1) {
    if (st + kLoraWaves < s1) load(f1, st + kLoraWaves);
    mma(f0);
    st += kLoraWaves;
    if (st >= s1) break;
    if (st + kLoraWaves < s1) load(f0, st + kLoraWaves);
    mma(f1);
    st += kLoraWaves;
  }
  // waves 2, 3 into 0, 1, then 1 into 0: half the LDS of four copies
  for (int half = kLoraWaves / 2; half > 0; half /= 2) {
    __syncthreads();
    if (w4 >= half && w4 < 2 * half) {
#pragma unroll
      for (int i = 0; i < MT * NT; ++i) red[w4 - half][i][lane] = acc[i / NT][i % NT];
    }
    __syncthreads();
    if (w4 < half) {
#pragma unroll
      for (int i = 0; i < MT * NT; ++i) acc[i / NT][i % NT] += red[w4][i][lane];
    }
  }
  if (w4) return;
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int row = i * 16 + 4 * q + e;
      if (row >= tile.rows) continue;
      float* p = h + ((int64_t)blockIdx.y * M + pos0 + row) * RP + rank0 + n16;
#pragma unroll
      for (int j = 0; j < NT; ++j) p[16 * j] = rank0 + 16 * j + n16 < r ? acc[i][j][e] : 0.f;
    }
}

// ---------------------------------------------------------------------------
// expand: out[src[pos]] = base[src[pos]] + s h[pos] . w[adapter]
// ---------------------------------------------------------------------------

// 8 ranks of a row of h, the splits added up in order.
__device__ __forceinline__ void load_h(const float* h, int S, int64_t stride, float (&v)[8]) {
  v4f a = *(const v4f*)h, b = *(const v4f*)(h + 4);
#pragma unroll 4
  for (int s = 1; s < S; ++s) {
    a += *(const v4f*)(h + s * stride);
    b += *(const v4f*)(h + s * stride + 4);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = a[i];
    v[4 + i] = b[i];
  }
}

// Workgroup: up to 64 tokens of one adapter, 16 a wave, by `chunks` times 128
// columns.  A wave adds up its tokens' rows of h and keeps them as operands in
// two terms; the 128 columns of the adapter come through LDS for all waves,
// the next ones on their way meanwhile.  A lane's sums are 8
// columns of 4 tokens, which meet base and output as 16-byte accesses, 256 bytes
// of a row together.  Ranks past 32 KS (BIG) are gone through 32 KS at a time,
// their rows of h read again for every column block.  The first columns'
// workgroups leave the added rows of h in hsum (if given) for the gradients.
// Workgroups past the tiles take the tokens without an adapter, 64 each: out =
// base (or 0).
template <typename T, int KS, bool BIG, bool ONCE>
__global__ __launch_bounds__(kLoraThreads, BIG ? 1 : KS == 4 ? 2 : 3) void lora_expand_kernel(
    const float* __restrict__ h, int S, int64_t M, int RP, const T* __restrict__ w, int64_t ldw_r, int64_t ldw_l, int r,
    int64_t N, const float* __restrict__ scales, const T* base, int64_t ldb, T* out, int64_t ldo,
    const int32_t* __restrict__ rows, int64_t tokens, const int32_t* __restrict__ src, const int32_t* __restrict__ offs,
    int L, int tiles, int chunks, int ranges, float* __restrict__ hsum) {
  constexpr int kRanks = 32 * KS, kStage = kRanks * 16 / kLoraThreads, kBufs = KS == 4 ? 1 : 2;
  constexpr bool kScaled = __is_same(T, _Float16);
  __shared__ v4u wbuf[kBufs][kRanks][17];            // 128 columns of a rank, and 16 bytes that spread the banks
  const int lane = threadIdx.x & (kWave - 1), n16 = lane & 15, q = lane >> 4, w4 = wave_id();
  const int t = blockIdx.x / ranges, cr = blockIdx.x - t * ranges;
  if (t >= tiles) {
    const int64_t t0 = (int64_t)(t - tiles) * kPassRows, end = (int64_t)(cr + 1) * chunks * kExpandCols;
    for (int i = w4; i < kPassRows; i += kLoraWaves) {
      if (t0 + i >= tokens || rows[t0 + i] >= 0) continue;
      for (int64_t col = (int64_t)cr * chunks * kExpandCols + lane * 8; col < end && col < N; col += 8 * kWave) {
        T v[8];
        const v4u b = base ? load8(base + (t0 + i) * ldb + col, N - col) : v4u{0, 0, 0, 0};
        __builtin_memcpy(v, &b, 16);
        store8<T, ONCE>(out + (t0 + i) * ldo + col, v, N - col);
      }
    }
    return;
  }
  const TileRoute tile = lora_tile<kExpandRows>(offs, L, t);
  if (tile.expert < 0) return;
  const int64_t pos0 = tile.start + (int64_t)tile.block * kExpandRows + w4 * 16;
  const int mine = tile.rows - w4 * 16;              // rows of this wave (past 16: of the next ones too)
  const bool in = n16 < mine;
  const float* hp = h + (pos0 + (in ? n16 : 0)) * RP + q * 8;
  const float scale = scales ? scales[tile.expert] : 1.f;
  int token[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) token[e] = 4 * q + e < mine ? src[pos0 + 4 * q + e] : -1;

  // weights: thread i takes 16 bytes i % 16 of ranks i / 16 + 16 k
  const T* wp = w + tile.expert * ldw_l;
  v4u stage[kStage];
  auto load_w = [&](int64_t col0, int rank0) {
    const int64_t col = col0 + (threadIdx.x & 15) * 8;
#pragma unroll
    for (int k = 0; k < kStage; ++k) {
      const int rank = rank0 + (int)(threadIdx.x >> 4) + 16 * k;
      stage[k] = rank < r ? load8(wp + (int64_t)rank * ldw_r + col, N - col) : v4u{0, 0, 0, 0};
    }
  };
  // column blocks: neighbouring tiles begin at different ones (rows a power of
  // two apart would have all of them at the same few memory channels)
  const int nb = BIG ? RP / kRanks : 1, first = cr * chunks;
  const int ncb = (int)((N + kExpandCols - 1) / kExpandCols), have = ncb - first < chunks ? ncb - first : chunks;
  auto column = [&](int i) { return (int64_t)(first + (i + t) % have) * kExpandCols; };
  load_w(column(0), 0);

  auto load_hidden = [&](int rank, float (&v)[8]) {
    if (in && rank + q * 8 < RP) {
      load_h(hp + rank, S, M * RP, v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.f;
    }
  };
  float up = 1.f, down = 1.f;
  auto set_scale = [&](uint32_t top) {               // of row n16, from its four lanes
    uint32_t o = (uint32_t)__shfl_xor((int)top, 16);
    top = o > top ? o : top;
    o = (uint32_t)__shfl_xor((int)top, 32);
    top = o > top ? o : top;
    up = row_scale(top, false);
    down = row_scale(top, true);
  };
  v4u hi[KS], lo[KS];
  if constexpr (!BIG) {
    float v[KS][8];
    uint32_t top = 0;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      load_hidden(ks * 32, v[ks]);
      if (hsum && cr == 0 && in && ks * 32 + q * 8 < RP) {
        float* p = hsum + (pos0 + n16) * RP + ks * 32 + q * 8;
        *(v4f*)p = v4f{v[ks][0], v[ks][1], v[ks][2], v[ks][3]};
        *(v4f*)(p + 4) = v4f{v[ks][4], v[ks][5], v[ks][6], v[ks][7]};
      }
      if (kScaled) top = top_bits(v[ks], top);
    }
    if (kScaled) set_scale(top);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[ks][i] *= down;
      two_terms<T>(v[ks], hi[ks], lo[ks]);
    }
  } else if (kScaled) {
    uint32_t top = 0;
    for (int rank = 0; rank < RP; rank += 32) {
      float v[8];
      load_hidden(rank, v);
      top = top_bits(v, top);
    }
    set_scale(top);
  }
  v4u old[4];
  v4f acc[8];
  int buf = 0;
  for (int i = 0; i < have * nb; ++i) {
    const int c = BIG ? i / nb : i, n = BIG ? i - c * nb : 0;
    if (kBufs == 1 && i > 0) __syncthreads();        // the block before has been read
#pragma unroll
    for (int k = 0; k < kStage; ++k) wbuf[buf][(threadIdx.x >> 4) + 16 * k][threadIdx.x & 15] = stage[k];
    __syncthreads();
    const bool more = i + 1 < have * nb;
    const int c1 = BIG ? (i + 1) / nb : i + 1;
    if (more) load_w(column(c1), BIG ? (i + 1 - c1 * nb) * kRanks : 0);
    const int64_t col = column(c) + 8 * n16, left = N - col;
    if (n == 0) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        old[e] = base && token[e] >= 0 ? load8<T, ONCE>(base + token[e] * ldb + col, left) : v4u{0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] = v4f{0.f, 0.f, 0.f, 0.f};
    }
    if (mine > 0) {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        if constexpr (BIG) {
          float v[8];
          load_hidden(n * kRanks + ks * 32, v);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] *= down;
          two_terms<T>(v, hi[ks], lo[ks]);
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {       // four columns of eight at a time: 16 registers fewer
          v2u row[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) row[j] = ((const v2u*)&wbuf[buf][ks * 32 + q * 8 + j][n16])[half];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const v4u b = column_of(row, j);
            acc[4 * half + j] = Mat<T>::mma(hi[ks], b, acc[4 * half + j]);
            acc[4 * half + j] = Mat<T>::mma(lo[ks], b, acc[4 * half + j]);
          }
        }
      }
      if (!BIG || n == nb - 1) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float f = kScaled ? scale * __shfl(up, 4 * q + e) : scale;
          if (token[e] < 0) continue;
          T o[8], y[8];
          __builtin_memcpy(o, &old[e], 16);
#pragma unroll
          for (int j = 0; j < 8; ++j) y[j] = (T)((float)o[j] + f * acc[j][e]);
          store8<T, ONCE>(out + token[e] * ldo + col, y, left);
        }
      }
    }
    buf = kBufs == 2 ? buf ^ 1 : 0;
  }
}

// The same for few tokens an adapter: workgroup of up to 16 tokens by 512
// columns, 128 a wave, the adapter straight from memory into operands.  Bound by
// the chain of loads (group ends, tokens, base) and the adapters' bytes: with the
// 64 x 128 tiles above, 64 tokens of as many adapters (rank 16, 8192 columns)
// took 13.6 us, four of the waves' places empty.
template <typename T>
__global__ __launch_bounds__(kLoraThreads) void lora_expand_few_kernel(
    const float* __restrict__ h, int S, int64_t M, int RP, const T* __restrict__ w, int64_t ldw_r, int64_t ldw_l, int r,
    int64_t N, const float* __restrict__ scales, const T* base, int64_t ldb, T* out, int64_t ldo,
    const int32_t* __restrict__ rows, int64_t tokens, const int32_t* __restrict__ src, const int32_t* __restrict__ offs,
    int L, int tiles, int ranges, float* __restrict__ hsum) {
  constexpr bool kScaled = __is_same(T, _Float16);
  const int lane = threadIdx.x & (kWave - 1), n16 = lane & 15, q = lane >> 4, w4 = wave_id();
  const int t = blockIdx.x / ranges, cr = blockIdx.x - t * ranges;
  const int64_t c0 = ((int64_t)cr * kLoraWaves + w4) * kExpandCols;
  if (c0 >= N) return;
  if (t >= tiles) {
    const int64_t t0 = (int64_t)(t - tiles) * 16 + q, col = c0 + 8 * n16;
    if (col >= N) return;
    for (int i = 0; i < 16; i += 4) {
      if (t0 + i >= tokens || rows[t0 + i] >= 0) continue;
      T v[8];
      const v4u b = base ? load8(base + (t0 + i) * ldb + col, N - col) : v4u{0, 0, 0, 0};
      __builtin_memcpy(v, &b, 16);
      store8(out + (t0 + i) * ldo + col, v, N - col);
    }
    return;
  }
  const TileRoute tile = lora_tile<16>(offs, L, t);
  if (tile.expert < 0) return;
  const int64_t pos0 = tile.start + (int64_t)tile.block * 16, col = c0 + 8 * n16, left = N - col;
  const bool in = n16 < tile.rows;
  const float* hp = h + (pos0 + (in ? n16 : 0)) * RP + q * 8;
  const T* wp = w + tile.expert * ldw_l + col;
  int token[4];
  v4u old[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) token[e] = 4 * q + e < tile.rows ? src[pos0 + 4 * q + e] : -1;
  float up = 1.f, down = 1.f;
  if (kScaled) {
    uint32_t top = 0;
    for (int rank = 0; rank + q * 8 < RP; rank += 32) {
      float v[8];
      load_h(hp + rank, S, M * RP, v);
      top = top_bits(v, top);
    }
    uint32_t o = (uint32_t)__shfl_xor((int)top, 16);
    top = o > top ? o : top;
    o = (uint32_t)__shfl_xor((int)top, 32);
    top = o > top ? o : top;
    up = row_scale(top, false);
    down = row_scale(top, true);
  }
  v4f acc[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) acc[j] = v4f{0.f, 0.f, 0.f, 0.f};
  for (int rank = 0; rank < RP; rank += 32) {
    v4u row[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int rr = rank + q * 8 + i;
      row[i] = rr < r ? load8(wp + (int64_t)rr * ldw_r, left) : v4u{0, 0, 0, 0};
    }
    float v[8];
    const bool have = in && rank + q * 8 < RP;
    if (have) {
      load_h(hp + rank, S, M * RP, v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.f;
    }
    if (hsum && cr == 0 && w4 == 0 && have) {
      float* p = hsum + (pos0 + n16) * RP + rank + q * 8;
      *(v4f*)p = v4f{v[0], v[1], v[2], v[3]};
      *(v4f*)(p + 4) = v4f{v[4], v[5], v[6], v[7]};
    }
    if (rank == 0) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        old[e] = base && token[e] >= 0 ? load8(base + token[e] * ldb + col, left) : v4u{0, 0, 0, 0};
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= down;
    v4u hi, lo;
    two_terms<T>(v, hi, lo);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const v4u b = column_of(row, j);
      acc[j] = Mat<T>::mma(hi, b, acc[j]);
      acc[j] = Mat<T>::mma(lo, b, acc[j]);
    }
  }
  const float scale = scales ? scales[tile.expert] : 1.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float f = kScaled ? scale * __shfl(up, 4 * q + e) : scale;
    if (token[e] < 0) continue;
    T o[8], y[8];
    __builtin_memcpy(o, &old[e], 16);
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = (T)((float)o[j] + f * acc[j][e]);
    store8(out + token[e] * ldo + col, y, left);
  }
}

// ---------------------------------------------------------------------------
// outer: gw[adapter][rank][col] = s sum over the adapter's tokens of h[pos][rank] x[src[pos]][col]
// ---------------------------------------------------------------------------

// One of the two gradients of a launch: h (M, RP) and x (T, K) to (L, r, K).
template <typename T>
struct Outer {
  const float* h;
  const T* x;
  int64_t ldx;
  int64_t K;          // 0: not asked for
  T* out;
};

__host__ __device__ __forceinline__ int outer_blocks(int64_t K) { return (int)((K + kOuterCols - 1) / kOuterCols); }

// Workgroup: 128 columns, 16 RT ranks and one chunk of an adapter's tokens,
// whose 32-token steps go round its four waves, joined in LDS.  With one chunk
// per adapter (part null) the result is stored, else the chunk's sums for
// lora_join_kernel: part (chunk, r, K of a + K of b).
template <typename T, int RT>
__global__ __launch_bounds__(kLoraThreads) void lora_outer_kernel(Outer<T> ga, Outer<T> gb, int RP, int r,
                                                                  const float* __restrict__ scales,
                                                                  const int32_t* __restrict__ src,
                                                                  const int32_t* __restrict__ offs, int L, int chunk,
                                                                  float* __restrict__ part) {
  constexpr int LD = kOuterCols + 4;
  __shared__ float red[kLoraWaves][16][LD];
  const int lane = threadIdx.x & (kWave - 1), n16 = lane & 15, q = lane >> 4, w4 = wave_id();
  const int na = outer_blocks(ga.K), ncb = na + outer_blocks(gb.K);
  const int t = blockIdx.x / ncb;
  int cb = blockIdx.x - t * ncb;
  const bool second = cb >= na;
  const Outer<T> g = second ? gb : ga;
  const int64_t shift = second ? ga.K : 0, wide = ga.K + gb.K;
  if (second) cb -= na;
  int adapter = t;
  int64_t lo, hi;
  if (part) {
    int pn;
    const TileRoute tile = route_tile(offs, L, chunk, 1, 1, t, pn);
    if (tile.expert < 0) return;
    adapter = tile.expert;
    lo = tile.start + (int64_t)tile.block * chunk;
    hi = lo + tile.rows;
  } else {
    lo = t > 0 ? offs[t - 1] : 0;
    hi = offs[t];
  }
  const int64_t col = (int64_t)cb * kOuterCols + 8 * n16, left = g.K - col;
  const int rank0 = blockIdx.y * 16 * RT;
  const float* hp = g.h + rank0 + n16;
  v4f acc[RT][8];
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
  for (int64_t p0 = lo + 32 * w4; p0 < hi; p0 += 32 * kLoraWaves) {
    int token[8];
    v4u row[8];
    float u[RT][8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t pos = p0 + 8 * q + i;
      token[i] = pos < hi ? src[pos] : -1;
#pragma unroll
      for (int a = 0; a < RT; ++a) u[a][i] = pos < hi ? hp[pos * RP + a * 16] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      row[i] = token[i] >= 0 ? load8(g.x + token[i] * g.ldx + col, left) : v4u{0, 0, 0, 0};
    v4u uh[RT], ul[RT];
#pragma unroll
    for (int a = 0; a < RT; ++a) {
#pragma unroll
      for (int i = 0; i < 8; ++i) u[a][i] = token[i] >= 0 ? u[a][i] : 0.f;   // a pad's row holds anything
      two_terms<__bf16>(u[a], uh[a], ul[a]);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v4u b = column_of(row, j);
      if constexpr (__is_same(T, _Float16)) {
        v4u bh, bl;
        two_terms_f16(b, bh, bl);
#pragma unroll
        for (int a = 0; a < RT; ++a) acc[a][j] = Mat<__bf16>::mma(uh[a], bl, acc[a][j]);
        b = bh;
      }
#pragma unroll
      for (int a = 0; a < RT; ++a) {
        acc[a][j] = Mat<__bf16>::mma(uh[a], b, acc[a][j]);
        acc[a][j] = Mat<__bf16>::mma(ul[a], b, acc[a][j]);
      }
    }
  }
  const float scale = scales ? scales[adapter] : 1.f;
#pragma unroll
  for (int a = 0; a < RT; ++a) {
    if (a) __syncthreads();
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int j = 0; j < 8; ++j) red[w4][4 * q + e][8 * n16 + j] = acc[a][j][e];
    __syncthreads();
    for (int e = threadIdx.x; e < 16 * kOuterCols; e += kLoraThreads) {
      const int rank = rank0 + a * 16 + e / kOuterCols;
      const int64_t c = (int64_t)cb * kOuterCols + e % kOuterCols;
      if (rank >= r || c >= g.K) continue;
      float v = 0.f;
#pragma unroll
      for (int i = 0; i < kLoraWaves; ++i) v += red[i][e / kOuterCols][e % kOuterCols];
      if (part)
        part[((int64_t)t * r + rank) * wide + shift + c] = v;
      else
        g.out[((int64_t)adapter * r + rank) * g.K + c] = (T)(scale * v);
    }
  }
}

// Adds up an adapter's chunks, in order, and rounds once; a workgroup takes 256
// columns of a rank of both gradients.
template <typename T>
__global__ __launch_bounds__(kLoraThreads) void lora_join_kernel(const float* __restrict__ part, Outer<T> ga, Outer<T> gb,
                                                                 int r, const float* __restrict__ scales,
                                                                 const int32_t* __restrict__ offs, int chunk) {
  const int a = blockIdx.z, rank = blockIdx.y;
  int first = 0, count = 0;
  for (int l0 = 0; l0 <= a; l0 += kWave) {           // chunks of the adapters before, and of this one
    const int l = l0 + (int)(threadIdx.x & (kWave - 1));
    int n = 0;
    if (l <= a) {
      const int rows = offs[l] - (l > 0 ? offs[l - 1] : 0);
      n = rows > 0 ? (rows + chunk - 1) / chunk : 0;
    }
    const int sum = wave_incl_scan(n);
    first += lane_value(sum, kWave - 1);
    if (a - l0 < kWave) count = lane_value(n, a - l0);
  }
  first -= count;
  const int64_t wide = ga.K + gb.K, c = (int64_t)blockIdx.x * kLoraThreads + threadIdx.x;
  if (c >= wide) return;
  const float* p = part + ((int64_t)first * r + rank) * wide + c;
  float v = 0.f;
#pragma unroll 8
  for (int i = 0; i < count; ++i) v += p[i * r * wide];
  v *= scales ? scales[a] : 1.f;
  if (c < ga.K)
    ga.out[((int64_t)a * r + rank) * ga.K + c] = (T)v;
  else
    gb.out[((int64_t)a * r + rank) * gb.K + c - ga.K] = (T)v;
}

// Adds up the splits of h (out may be the first).
__global__ __launch_bounds__(kLoraThreads) void lora_sum_kernel(const float* h, int S, int64_t n, float* out) {
  const int64_t i = ((int64_t)blockIdx.x * kLoraThreads + threadIdx.x) * 8;
  if (i >= n) return;
  float v[8];
  load_h(h + i, S, n, v);
  *(v4f*)(out + i) = v4f{v[0], v[1], v[2], v[3]};
  *(v4f*)(out + i + 4) = v4f{v[4], v[5], v[6], v[7]};
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

static int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Ranks as shrink computes them and h holds them: 16, 32, 64 or multiples of 128.
static int rank_pad(int r) { return r <= 16 ? 16 : r <= 32 ? 32 : r <= 64 ? 64 : (int)cdiv(r, 128) * 128; }

// Fewer than 32 tokens an adapter on average: tiles of 16 token rows.
static bool few_tokens(int64_t M, int L) { return M < 32 * (int64_t)L; }

// Token rows of a shrink tile: 64 (32 beside 128 ranks), or 16.
static int shrink_rows(int64_t M, int L, int r) { return few_tokens(M, L) ? 16 : r > 64 ? 32 : 64; }

static int shrink_splits(int64_t M, int L, int r, int64_t K) {
  const int64_t used = M < L ? M : L, tiles = cdiv(M, shrink_rows(M, L, r)) + used / 2;
  const int64_t want = cdiv(1024, tiles > 0 ? tiles * cdiv(rank_pad(r), 128) : 1), most = cdiv(K, 64 * 2 * kLoraWaves);
  const int64_t s = want < most ? want : most;
  return (int)(s < 1 ? 1 : s > 8 ? 8 : s);
}

// Tokens of an outer chunk (columns K of both gradients together): enough
// chunks for 1024 workgroups, 256 tokens at least.
static int outer_chunk(int64_t M, int64_t K) {
  const int64_t c = cdiv(M * cdiv(K, kOuterCols), 1024 * 32) * 32;
  return (int)(c < 256 ? 256 : c);
}

// f32 of the chunks' sums; 0 where every adapter is one chunk.
static int64_t outer_floats(int64_t M, int L, int r, int64_t K) {
  const int chunk = outer_chunk(M, K);
  return M <= chunk ? 0 : (cdiv(M, chunk) + (M < L ? M : L)) * r * K;
}

static int lora_args(const char* what, int dtype, int r, int L, int64_t M, int64_t K, int64_t N) {
  if (dtype != MXGG_DTYPE_BF16 && dtype != MXGG_DTYPE_F16)
    return fail(MXGG_ERR_INVALID_ARG, "%s: element type %d is neither bf16 nor f16", what, dtype);
  if (r < 1 || r > kMaxRank) return fail(MXGG_ERR_INVALID_ARG, "%s: rank %d, expected 1 to %d", what, r, kMaxRank);
  if (L < 1 || L > kMaxAdapters) return fail(MXGG_ERR_INVALID_ARG, "%s: %d adapters, expected 1 to %d", what, L, kMaxAdapters);
  if (M < 0 || M > 0x7fffffffll - kMaxAdapters || K < 1 || K > (1ll << 30) || N < 1 || N > (1ll << 30))
    return fail(MXGG_ERR_INVALID_ARG, "%s: %lld rows of %lld and %lld elements are out of range", what, (long long)M,
                (long long)K, (long long)N);
  return MXGG_OK;
}

template <typename T>
static int launch_shrink(const void* x, int64_t ldx, int64_t K, const void* w, int64_t ldw_r, int64_t ldw_l, int r,
                         const int32_t* src, const int32_t* offs, int L, int64_t M, float* h, int S, hipStream_t st) {
  const int rows = shrink_rows(M, L, r), RP = rank_pad(r);
  const dim3 grid((unsigned)(cdiv(M, rows) + (M < L ? M : L)), S, RP > 128 ? RP / 128 : 1);
#define MXGG_SHRINK(MT, NT)                                                                                    \
  lora_shrink_kernel<T, MT, NT><<<grid, kLoraThreads, 0, st>>>((const T*)x, ldx, K, (const T*)w, ldw_r, ldw_l, r, src, \
                                                               offs, L, M, h, RP)
  if (rows == 16) {
    if (RP == 16) MXGG_SHRINK(1, 1);
    else if (RP == 32) MXGG_SHRINK(1, 2);
    else if (RP == 64) MXGG_SHRINK(1, 4);
    else MXGG_SHRINK(1, 8);
  } else {
    if (RP == 16) MXGG_SHRINK(4, 1);
    else if (RP == 32) MXGG_SHRINK(4, 2);
    else if (RP == 64) MXGG_SHRINK(4, 4);
    else MXGG_SHRINK(2, 8);
  }
#undef MXGG_SHRINK
  return launch_status("lora_shrink_kernel");
}

static int launch_sum(const float* h, int S, int64_t n, float* out, hipStream_t st) {
  lora_sum_kernel<<<(unsigned)cdiv(n, 8 * kLoraThreads), kLoraThreads, 0, st>>>(h, S, n, out);
  return launch_status("lora_sum_kernel");
}

template <typename T>
static int launch_expand(float* h, int S, int64_t M, const void* w, int64_t ldw_r, int64_t ldw_l, int r, int64_t N,
                         const float* scales, const void* base, int64_t ldb, void* out, int64_t ldo,
                         const int32_t* rows, int64_t tokens, const int32_t* src, const int32_t* offs, int L,
                         float* hsum, hipStream_t st) {
  const int RP = rank_pad(r);
  if (few_tokens(M, L)) {
    const int64_t used = M < L ? M : L, tiles = cdiv(M, 16) + used, none = base == out ? 0 : cdiv(tokens, 16);
    const int64_t ranges = cdiv(N, kLoraWaves * kExpandCols), grid = (tiles + none) * ranges;
    if (grid > 0xffffff) return fail(MXGG_ERR_INVALID_ARG, "lora_expand: too large");
    lora_expand_few_kernel<T><<<(unsigned)grid, kLoraThreads, 0, st>>>(
        h, S, M, RP, (const T*)w, ldw_r, ldw_l, r, N, scales, (const T*)base, ldb, (T*)out, ldo, rows, tokens, src, offs,
        L, (int)tiles, (int)ranges, hsum);
    return launch_status("lora_expand_few_kernel");
  }
  if (RP > 128 && (S > 1 || hsum)) {                 // h is read for every column block: added up once
    float* sum = hsum ? hsum : h;
    if (int rc = launch_sum(h, S, M * RP, sum, st)) return rc;
    h = sum;
    S = 1;
    hsum = nullptr;
  }
  const int64_t used = M < L ? M : L, tiles = cdiv(M, kExpandRows) + used;
  const int64_t none = base == out ? 0 : cdiv(tokens, kPassRows), ncb = cdiv(N, kExpandCols);
  // column blocks of a workgroup: four where that leaves 1024 workgroups (16640
  // tokens, rank 64, 8192 columns: one 202 us, two 146, four 125, sixteen 145;
  // long workgroups lose the order in which memory likes to be read)
  int64_t chunks = (cdiv(M, kExpandRows) + used / 2) * ncb / 1024;
  chunks = chunks < 1 ? 1 : chunks > 4 ? 4 : chunks;
  const int64_t ranges = cdiv(ncb, chunks), grid = (tiles + none) * ranges;
  if (grid > 0xffffff) return fail(MXGG_ERR_INVALID_ARG, "lora_expand: too large");
  const bool once = tokens * N * (int64_t)sizeof(T) > (32ll << 20);
#define MXGG_EXPAND(KS, BIG) (once ? lora_expand_kernel<T, KS, BIG, true> : lora_expand_kernel<T, KS, BIG, false>)
  const auto kernel = RP <= 32    ? MXGG_EXPAND(1, false)
                      : RP == 64  ? MXGG_EXPAND(2, false)
                      : RP == 128 ? MXGG_EXPAND(4, false)
                                  : MXGG_EXPAND(4, true);
#undef MXGG_EXPAND
  kernel<<<(unsigned)grid, kLoraThreads, 0, st>>>(h, S, M, RP, (const T*)w, ldw_r, ldw_l, r, N, scales, (const T*)base,
                                                  ldb, (T*)out, ldo, rows, tokens, src, offs, L, (int)tiles, (int)chunks,
                                                  (int)ranges, hsum);
  return launch_status("lora_expand_kernel");
}

template <typename T>
static int launch_outer(const Outer<T>& ga, const Outer<T>& gb, int64_t M, int r, const float* scales, const int32_t* src,
                        const int32_t* offs, int L, float* part, hipStream_t st) {
  const int64_t K = ga.K + gb.K, ncb = outer_blocks(ga.K) + outer_blocks(gb.K);
  const int RP = rank_pad(r), chunk = outer_chunk(M, K);
  const bool one = M <= chunk;
  const int64_t tiles = one ? L : cdiv(M, chunk) + (M < L ? M : L);
  if (tiles * ncb > 0xffffff) return fail(MXGG_ERR_INVALID_ARG, "lora_grouped_mm_grad: too large");
  const int rt = RP == 16 ? 1 : RP == 32 ? 2 : 4;
  const auto kernel = rt == 1 ? lora_outer_kernel<T, 1> : rt == 2 ? lora_outer_kernel<T, 2> : lora_outer_kernel<T, 4>;
  kernel<<<dim3((unsigned)(tiles * ncb), RP / (16 * rt)), kLoraThreads, 0, st>>>(ga, gb, RP, r, scales, src, offs, L,
                                                                                chunk, one ? nullptr : part);
  int rc = launch_status("lora_outer_kernel");
  if (rc != MXGG_OK || one) return rc;
  lora_join_kernel<T><<<dim3((unsigned)cdiv(K, kLoraThreads), r, L), kLoraThreads, 0, st>>>(part, ga, gb, r, scales, offs,
                                                                                           chunk);
  return launch_status("lora_join_kernel");
}

// Places of the gradients' workspace (f32, 256-byte steps): u's splits, their
// sum, the chunks' sums of outer.
struct GradRoom {
  int64_t u, usum, part, total;
};

static GradRoom grad_room(int64_t M, int L, int r, int64_t K, int64_t N) {
  auto up = [](int64_t n) { return cdiv(n, 64) * 64; };
  const int64_t row = up(M * rank_pad(r)), both = outer_floats(M, L, r, K + N), one = outer_floats(M, L, r, K),
                other = outer_floats(M, L, r, N), part = both > one ? (both > other ? both : other) : one > other ? one : other;
  GradRoom g{0, 0, 0, 0};
  g.usum = up((int64_t)shrink_splits(M, L, r, N) * M * rank_pad(r));
  g.part = g.usum + row;
  g.total = g.part + part;
  return g;
}

struct LoraGrad {
  const void *x, *down, *up, *g;
  int64_t ldx, ldd_r, ldd_l, ldu_r, ldu_l, ldg;
  const float *h, *scales;
  const int32_t *rows, *src, *offs;
  int64_t tokens, M, K, N;
  int r, L;
  void *gx, *gdown, *gup;
  float* ws;
};

template <typename T>
static int launch_grad(const LoraGrad& a, hipStream_t st) {
  const GradRoom room = grad_room(a.M, a.L, a.r, a.K, a.N);
  float *u = a.ws + room.u, *usum = a.ws + room.usum, *part = a.ws + room.part;
  const int S = shrink_splits(a.M, a.L, a.r, a.N);
  if (a.gx || a.gdown) {
    if (int rc = launch_shrink<T>(a.g, a.ldg, a.N, a.up, a.ldu_r, a.ldu_l, a.r, a.src, a.offs, a.L, a.M, u, S, st)) return rc;
  }
  if (a.gx) {
    if (int rc = launch_expand<T>(u, S, a.M, a.down, a.ldd_r, a.ldd_l, a.r, a.K, a.scales, nullptr, 0, a.gx, a.K, a.rows,
                                  a.tokens, a.src, a.offs, a.L, usum, st))
      return rc;
  } else if (a.gdown) {
    if (int rc = launch_sum(u, S, a.M * rank_pad(a.r), usum, st)) return rc;
  }
  if (!a.gdown && !a.gup) return MXGG_OK;
  const Outer<T> ga{usum, (const T*)a.x, a.ldx, a.gdown ? a.K : 0, (T*)a.gdown};
  const Outer<T> gb{a.h, (const T*)a.g, a.ldg, a.gup ? a.N : 0, (T*)a.gup};
  return launch_outer<T>(ga, gb, a.M, a.r, a.scales, a.src, a.offs, a.L, part, st);
}

}  // namespace mxgg

using namespace mxgg;

extern "C" int64_t mxgg_lora_hidden_floats(int64_t M, int r) {
  return M < 1 || r < 1 || r > kMaxRank ? 0 : M * rank_pad(r);
}

extern "C" int64_t mxgg_lora_workspace_floats(int64_t M, int L, int r, int64_t K) {
  return M < 1 || L < 1 || r < 1 || r > kMaxRank || K < 1 ? 0 : (int64_t)shrink_splits(M, L, r, K) * M * rank_pad(r);
}

extern "C" int64_t mxgg_lora_grad_workspace_floats(int64_t M, int L, int r, int64_t K, int64_t N) {
  return M < 1 || L < 1 || r < 1 || r > kMaxRank || K < 1 || N < 1 ? 0 : grad_room(M, L, r, K, N).total;
}

extern "C" int mxgg_lora_grouped_mm(const void* x, int dtype, int64_t tokens, int64_t K, int64_t ldx, const void* down,
                                    int64_t ldd_r, int64_t ldd_l, const void* up, int64_t N, int64_t ldu_r,
                                    int64_t ldu_l, int r, const float* scales, const void* base, int64_t ldb, void* out,
                                    int64_t ldo, const int32_t* rows, const int32_t* src, const int32_t* offs, int L,
                                    int64_t M, float* hidden, float* workspace, int64_t ws_floats, void* stream) {
  clear_error();
  if (int rc = lora_args("lora_grouped_mm", dtype, r, L, M, K, N)) return rc;
  if (tokens < 0 || tokens > M) return fail(MXGG_ERR_INVALID_ARG, "lora_grouped_mm: %lld tokens in a plan of %lld rows", (long long)tokens, (long long)M);
  if (tokens == 0) return MXGG_OK;
  if (!x || !down || !up || !out || !rows || !src || !offs) return fail(MXGG_ERR_INVALID_ARG, "lora_grouped_mm: null pointer");
  if ((r > 1 && (ldd_r < K || ldu_r < N)) || (tokens > 1 && (ldx < K || ldo < N || (base && ldb < N))))
    return fail(MXGG_ERR_INVALID_ARG, "lora_grouped_mm: row stride below the row (K=%lld, N=%lld)", (long long)K, (long long)N);
  const int64_t need = mxgg_lora_workspace_floats(M, L, r, K);
  if (!workspace || ws_floats < need)
    return fail(MXGG_ERR_WORKSPACE, "lora_grouped_mm: workspace of %lld floats needed", (long long)need);
  if (int rc = require_device()) return rc;
  const int S = shrink_splits(M, L, r, K);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == MXGG_DTYPE_BF16) {
    if (int rc = launch_shrink<__bf16>(x, ldx, K, down, ldd_r, ldd_l, r, src, offs, L, M, workspace, S, st)) return rc;
    return launch_expand<__bf16>(workspace, S, M, up, ldu_r, ldu_l, r, N, scales, base, ldb, out, ldo, rows, tokens, src,
                                 offs, L, hidden, st);
  }
  if (int rc = launch_shrink<_Float16>(x, ldx, K, down, ldd_r, ldd_l, r, src, offs, L, M, workspace, S, st)) return rc;
  return launch_expand<_Float16>(workspace, S, M, up, ldu_r, ldu_l, r, N, scales, base, ldb, out, ldo, rows, tokens, src,
                                 offs, L, hidden, st);
}

extern "C" int mxgg_lora_grouped_mm_grad(const void* g, int dtype, int64_t tokens, int64_t ldg, const void* x, int64_t K,
                                         int64_t ldx, const void* down, int64_t ldd_r, int64_t ldd_l, const void* up,
                                         int64_t N, int64_t ldu_r, int64_t ldu_l, int r, const float* scales,
                                         const float* hidden, const int32_t* rows, const int32_t* src,
                                         const int32_t* offs, int L, int64_t M, void* g_x, void* g_down, void* g_up,
                                         float* workspace, int64_t ws_floats, void* stream) {
  clear_error();
  if (int rc = lora_args("lora_grouped_mm_grad", dtype, r, L, M, K, N)) return rc;
  if (tokens < 1 || tokens > M) return fail(MXGG_ERR_INVALID_ARG, "lora_grouped_mm_grad: %lld tokens in a plan of %lld rows", (long long)tokens, (long long)M);
  if (!g || !x || !down || !up || !rows || !src || !offs || (g_up && !hidden))
    return fail(MXGG_ERR_INVALID_ARG, "lora_grouped_mm_grad: null pointer");
  if ((r > 1 && (ldd_r < K || ldu_r < N)) || (tokens > 1 && (ldx < K || ldg < N)))
    return fail(MXGG_ERR_INVALID_ARG, "lora_grouped_mm_grad: row stride below the row (K=%lld, N=%lld)", (long long)K, (long long)N);
  const int64_t need = mxgg_lora_grad_workspace_floats(M, L, r, K, N);
  if (!workspace || ws_floats < need)
    return fail(MXGG_ERR_WORKSPACE, "lora_grouped_mm_grad: workspace of %lld floats needed", (long long)need);
  if (int rc = require_device()) return rc;
  const LoraGrad a{x, down, up, g, ldx, ldd_r, ldd_l, ldu_r, ldu_l, ldg, hidden, scales, rows, src, offs, tokens, M, K, N,
                   r, L, g_x, g_down, g_up, workspace};
  return dtype == MXGG_DTYPE_BF16 ? launch_grad<__bf16>(a, (hipStream_t)stream) : launch_grad<_Float16>(a, (hipStream_t)stream);
}
