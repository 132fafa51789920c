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

constexpr int kLoraThreads = 256;
constexpr int kLoraWaves = kLoraThreads / kWave;
constexpr int kMaxRank = 512;
constexpr int kMaxAdapters = 1024;
constexpr int kExpandRows = 64;      // token rows of an expand workgroup
constexpr int kExpandCols = 512;     // and its columns, 128 a wave
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
template <typename T>
__device__ __forceinline__ v4u load8(const T* p, int64_t left) {
  v4u r;
  if (left >= 8) {
    r = load_any(p);
  } else {
    T v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < left ? p[i] : (T)0.f;
    __builtin_memcpy(&r, v, 16);
  }
  return r;
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const T (&v)[8], int64_t left) {
  if (left >= 8) {
    v4u r;
    __builtin_memcpy(&r, v, 16);
    store_any(p, r);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) p[i] = v[i];
  }
}

// Operand j of 8 from 8 rows of 8 16-bit columns: column j of all rows.
__device__ __forceinline__ v4u column_of(const v4u (&row)[8], int j) {
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
__global__ __launch_bounds__(kLoraThreads) void lora_shrink_kernel(const T* __restrict__ x, int64_t ldx, int64_t K,
                                                                   const T* __restrict__ w, int64_t ldw_r,
                                                                   int64_t ldw_l, int r,
                                                                   const int32_t* __restrict__ src,
                                                                   const int32_t* __restrict__ offs, int L, int64_t M,
                                                                   float* __restrict__ h, int RP) {
  constexpr int BM = 16 * MT, BN = 16 * NT, LD = BN + 4;
  __shared__ float red[kLoraWaves][BM][LD];
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
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) red[w4][i * 16 + 4 * q + e][j * 16 + n16] = acc[i][j][e];
  __syncthreads();
  for (int e = threadIdx.x; e < BM * BN; e += kLoraThreads) {
    const int row = e / BN, col = e % BN;
    if (row >= tile.rows) continue;
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < kLoraWaves; ++i) v += red[i][row][col];
    h[((int64_t)blockIdx.y * M + pos0 + row) * RP + rank0 + col] = rank0 + col < r ? v : 0.f;
  }
}

// ---------------------------------------------------------------------------
// expand: out[src[pos]] = base[src[pos]] + s h[pos] . w[adapter]
// ---------------------------------------------------------------------------

// 8 ranks of a row of h, the splits added up.
__device__ __forceinline__ void load_h(const float* __restrict__ h, int S, int64_t stride, float (&v)[8]) {
  v4f a = *(const v4f*)h, b = *(const v4f*)(h + 4);
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

// Workgroup: up to 64 tokens of one adapter by 512 columns, 128 a wave.  A
// wave holds its columns of the adapter (32 KS ranks) as operands and goes over
// the tokens 16 at a time; the sums' 8 columns a lane meet base and the output
// as 16-byte accesses, 256 bytes of a row together.  Workgroups past the tiles
// take the tokens without an adapter, 64 each: out = base (or 0).
template <typename T, int KS>
__global__ __launch_bounds__(kLoraThreads) void lora_expand_kernel(const float* __restrict__ h, int S, int64_t M, int RP,
                                                                   const T* __restrict__ w, int64_t ldw_r,
                                                                   int64_t ldw_l, int r, int64_t N,
                                                                   const float* __restrict__ scales,
                                                                   const T* base, int64_t ldb, T* out, int64_t ldo,
                                                                   const int32_t* __restrict__ rows, int64_t tokens,
                                                                   const int32_t* __restrict__ src,
                                                                   const int32_t* __restrict__ offs, int L, int tiles) {
  const int lane = threadIdx.x & (kWave - 1), n16 = lane & 15, q = lane >> 4, w4 = wave_id();
  const int ncb = (int)((N + kExpandCols - 1) / kExpandCols);
  const int t = blockIdx.x / ncb, cb = blockIdx.x % ncb;
  if (t >= tiles) {
    const int64_t col = (int64_t)cb * kExpandCols + lane * 8, t0 = (int64_t)(t - tiles) * kExpandRows;
    for (int i = w4; i < kExpandRows; i += kLoraWaves) {
      if (t0 + i >= tokens || rows[t0 + i] >= 0 || col >= N) continue;
      T v[8];
      const v4u b = base ? load8(base + (t0 + i) * ldb + col, N - col) : v4u{0, 0, 0, 0};
      __builtin_memcpy(v, &b, 16);
      store8(out + (t0 + i) * ldo + col, v, N - col);
    }
    return;
  }
  const TileRoute tile = lora_tile<kExpandRows>(offs, L, t);
  const int64_t c0 = (int64_t)cb * kExpandCols + w4 * 128, col = c0 + 8 * n16, left = N - col;
  if (tile.expert < 0 || c0 >= N) return;
  const int64_t pos0 = tile.start + (int64_t)tile.block * kExpandRows;
  const float scale = scales ? scales[tile.expert] : 1.f;
  const T* wp = w + tile.expert * ldw_l + col;
  v4u b[KS][8];
  auto load_w = [&](int rank0) {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      v4u row[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int rank = rank0 + ks * 32 + q * 8 + i;
        row[i] = rank < r ? load8(wp + (int64_t)rank * ldw_r, left) : v4u{0, 0, 0, 0};
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) b[ks][j] = column_of(row, j);
    }
  };
  load_w(0);
  for (int sub = 0; sub < tile.rows; sub += 16) {
    const int row = sub + n16;
    const bool in = row < tile.rows;
    const float* hp = h + (pos0 + (in ? row : 0)) * RP + q * 8;
    int token[4];
    v4u old[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int rr = sub + 4 * q + e;
      token[e] = rr < tile.rows ? src[pos0 + rr] : -1;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      old[e] = base && token[e] >= 0 ? load8(base + token[e] * ldb + col, left) : v4u{0, 0, 0, 0};
    // f16: the row as 2^e times values below 2, so that neither term leaves the type
    float up = 1.f, down = 1.f;
    if constexpr (sizeof(T) == 2 && __is_same(T, _Float16)) {
      float m = 0.f;
      for (int k = q * 8; k < RP; k += 32) {
        float v[8];
        load_h(hp + (k - q * 8), S, M * RP, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(v[i]));
      }
      m = fmaxf(m, __shfl_xor(m, 16));
      m = fmaxf(m, __shfl_xor(m, 32));
      if (m > 0x1p-120f && m < 0x1p120f) {
        const uint32_t e = __float_as_uint(m) & 0x7f800000u;
        up = __uint_as_float(e);
        down = __uint_as_float(0x7f000000u - e);
      }
    }
    v4f acc[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] = v4f{0.f, 0.f, 0.f, 0.f};
    for (int rank0 = 0; rank0 < RP; rank0 += 32 * KS) {
      if (RP > 32 * KS && (rank0 > 0 || sub > 0)) load_w(rank0);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        float v[8];
        if (in && rank0 + ks * 32 + q * 8 < RP) {
          load_h(hp + rank0 + ks * 32, S, M * RP, v);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= down;
        v4u hi, lo;
        two_terms<T>(v, hi, lo);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          acc[j] = Mat<T>::mma(hi, b[ks][j], acc[j]);
          acc[j] = Mat<T>::mma(lo, b[ks][j], acc[j]);
        }
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float f = scale * __shfl(up, 4 * q + e);
      if (token[e] < 0) continue;
      T o[8], v[8];
      __builtin_memcpy(o, &old[e], 16);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = (T)((float)o[j] + f * acc[j][e]);
      store8(out + token[e] * ldo + col, v, left);
    }
  }
}

// ---------------------------------------------------------------------------
// outer: gw[adapter][rank][col] = s sum over the adapter's tokens of h[pos][rank] x[src[pos]][col]
// ---------------------------------------------------------------------------

// Workgroup: 128 columns, 16 RT ranks and one chunk of an adapter's tokens,
// whose 32-token steps go round its four waves, joined in LDS.  With one chunk
// per adapter (part null) the result is stored, else the chunk's sums (slot =
// chunk) for lora_join_kernel.
template <typename T, int RT>
__global__ __launch_bounds__(kLoraThreads) void lora_outer_kernel(const float* __restrict__ h, int S, int64_t M, int RP,
                                                                  int r, const T* __restrict__ x, int64_t ldx,
                                                                  int64_t K, const float* __restrict__ scales,
                                                                  const int32_t* __restrict__ src,
                                                                  const int32_t* __restrict__ offs, int L, int chunk,
                                                                  T* __restrict__ out, float* __restrict__ part) {
  constexpr int LD = kOuterCols + 4;
  __shared__ float red[kLoraWaves][16][LD];
  const int lane = threadIdx.x & (kWave - 1), n16 = lane & 15, q = lane >> 4, w4 = wave_id();
  const int ncb = (int)((K + kOuterCols - 1) / kOuterCols);
  const int t = blockIdx.x / ncb, cb = blockIdx.x % ncb;
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
  const int64_t col = (int64_t)cb * kOuterCols + 8 * n16, left = K - col;
  const int rank0 = blockIdx.y * 16 * RT;
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
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      row[i] = token[i] >= 0 ? load8(x + token[i] * ldx + col, left) : v4u{0, 0, 0, 0};
#pragma unroll
    for (int a = 0; a < RT; ++a)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float v = 0.f;
        if (token[i] >= 0) {
          const float* hp = h + (p0 + 8 * q + i) * RP + rank0 + a * 16 + n16;
          v = hp[0];
          for (int s = 1; s < S; ++s) v += hp[s * M * RP];
        }
        u[a][i] = v;
      }
    v4u uh[RT], ul[RT];
#pragma unroll
    for (int a = 0; a < RT; ++a) two_terms<__bf16>(u[a], uh[a], ul[a]);
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
      if (rank >= r || c >= K) continue;
      float v = 0.f;
#pragma unroll
      for (int i = 0; i < kLoraWaves; ++i) v += red[i][e / kOuterCols][e % kOuterCols];
      if (part)
        part[((int64_t)t * r + rank) * K + c] = v;
      else
        out[((int64_t)adapter * r + rank) * K + c] = (T)(scale * v);
    }
  }
}

// Adds up an adapter's chunks, in order, and rounds once.
template <typename T>
__global__ __launch_bounds__(kLoraThreads) void lora_join_kernel(const float* __restrict__ part, int r, int64_t K,
                                                                 const float* __restrict__ scales,
                                                                 const int32_t* __restrict__ offs, int chunk,
                                                                 T* __restrict__ out) {
  const int a = blockIdx.y;
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
  const int64_t size = r * K, i = (int64_t)blockIdx.x * kLoraThreads + threadIdx.x;
  if (i >= size) return;
  float v = 0.f;
#pragma unroll 4
  for (int c = 0; c < count; ++c) v += part[(first + c) * size + i];
  out[a * size + i] = (T)((scales ? scales[a] : 1.f) * v);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

static int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Ranks as shrink computes them and h holds them: 16, 32, 64 or multiples of 128.
static int rank_pad(int r) { return r <= 16 ? 16 : r <= 32 ? 32 : r <= 64 ? 64 : (int)cdiv(r, 128) * 128; }

// Token rows of a shrink tile: 64 (32 beside 128 ranks) where the adapters have
// that many tokens on average, else 16.
static int shrink_rows(int64_t M, int L, int r) { return M < 32 * (int64_t)L ? 16 : r > 64 ? 32 : 64; }

static int shrink_splits(int64_t M, int L, int r, int64_t K) {
  const int64_t used = M < L ? M : L, tiles = cdiv(M, shrink_rows(M, L, r)) + used / 2;
  const int64_t want = cdiv(1024, tiles > 0 ? tiles * cdiv(rank_pad(r), 128) : 1), most = cdiv(K, 64 * 2 * kLoraWaves);
  const int64_t s = want < most ? want : most;
  return (int)(s < 1 ? 1 : s > 32 ? 32 : s);
}

// Tokens of an outer chunk: enough chunks for 1024 workgroups, 256 tokens at least.
static int outer_chunk(int64_t M, int64_t K) {
  const int64_t c = cdiv(M * cdiv(K, kOuterCols), 1024 * 32) * 32;
  return (int)(c < 256 ? 256 : c);
}

static int lora_args(const char* what, int dtype, int r, int L, int64_t M, int64_t K) {
  if (dtype != MXGG_DTYPE_BF16 && dtype != MXGG_DTYPE_F16)
    return fail(MXGG_ERR_INVALID_ARG, "%s: element type %d is neither bf16 nor f16", what, dtype);
  if (r < 1 || r > kMaxRank) return fail(MXGG_ERR_INVALID_ARG, "%s: rank %d, expected 1 to %d", what, r, kMaxRank);
  if (L < 1 || L > kMaxAdapters) return fail(MXGG_ERR_INVALID_ARG, "%s: %d adapters, expected 1 to %d", what, L, kMaxAdapters);
  if (M < 0 || M > 0x7fffffffll - kMaxAdapters || K < 1 || K > (1ll << 30))
    return fail(MXGG_ERR_INVALID_ARG, "%s: %lld rows of %lld elements are out of range", what, (long long)M, (long long)K);
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

template <typename T>
static int launch_expand(const float* h, int S, int64_t M, const void* w, int64_t ldw_r, int64_t ldw_l, int r, int64_t N,
                         const float* scales, const void* base, int64_t ldb, void* out, int64_t ldo,
                         const int32_t* rows, int64_t tokens, const int32_t* src, const int32_t* offs, int L,
                         hipStream_t st) {
  const int RP = rank_pad(r);
  const int64_t tiles = cdiv(M, kExpandRows) + (M < L ? M : L), none = base == out ? 0 : cdiv(tokens, kExpandRows);
  const int64_t grid = (tiles + none) * cdiv(N, kExpandCols);
  if (grid > 0x7fffffffll) return fail(MXGG_ERR_INVALID_ARG, "lora_expand: too large");
  const auto kernel = RP <= 32 ? lora_expand_kernel<T, 1> : RP == 64 ? lora_expand_kernel<T, 2> : lora_expand_kernel<T, 4>;
  kernel<<<(unsigned)grid, kLoraThreads, 0, st>>>(h, S, M, RP, (const T*)w, ldw_r, ldw_l, r, N, scales, (const T*)base,
                                                  ldb, (T*)out, ldo, rows, tokens, src, offs, L, (int)tiles);
  return launch_status("lora_expand_kernel");
}

template <typename T>
static int launch_outer(const float* h, int S, int64_t M, int r, const void* x, int64_t ldx, int64_t K,
                        const float* scales, const int32_t* src, const int32_t* offs, int L, void* out, float* part,
                        hipStream_t st) {
  const int RP = rank_pad(r), chunk = outer_chunk(M, K);
  const bool one = M <= chunk;
  const int64_t tiles = one ? L : cdiv(M, chunk) + (M < L ? M : L), ncb = cdiv(K, kOuterCols);
  if (tiles * ncb > 0x7fffffffll) return fail(MXGG_ERR_INVALID_ARG, "lora_outer: too large");
  const int rt = RP == 16 ? 1 : RP == 32 ? 2 : 4;
  const dim3 grid((unsigned)(tiles * ncb), RP / (16 * rt));
  const auto kernel = rt == 1 ? lora_outer_kernel<T, 1> : rt == 2 ? lora_outer_kernel<T, 2> : lora_outer_kernel<T, 4>;
  kernel<<<grid, kLoraThreads, 0, st>>>(h, S, M, RP, r, (const T*)x, ldx, K, scales, src, offs, L, chunk, (T*)out,
                                        one ? nullptr : part);
  int rc = launch_status("lora_outer_kernel");
  if (rc != MXGG_OK || one) return rc;
  lora_join_kernel<T><<<dim3((unsigned)cdiv(r * K, kLoraThreads), L), kLoraThreads, 0, st>>>(part, r, K, scales, offs,
                                                                                            chunk, (T*)out);
  return launch_status("lora_join_kernel");
}

}  // namespace mxgg

using namespace mxgg;

extern "C" int64_t mxgg_lora_hidden_floats(int64_t M, int L, int r, int64_t K) {
  if (M < 1 || L < 1 || r < 1 || r > kMaxRank || K < 1) return 0;
  return (int64_t)shrink_splits(M, L, r, K) * M * rank_pad(r);
}

extern "C" int64_t mxgg_lora_outer_floats(int64_t M, int L, int r, int64_t K) {
  if (M < 1 || L < 1 || r < 1 || r > kMaxRank || K < 1) return 0;
  const int chunk = outer_chunk(M, K);
  return M <= chunk ? 0 : (cdiv(M, chunk) + (M < L ? M : L)) * r * K;
}

extern "C" int mxgg_lora_shrink(const void* x, int dtype, int64_t K, int64_t ldx, const void* w, int64_t ldw_r,
                                int64_t ldw_l, int r, const int32_t* src, const int32_t* offs, int L, int64_t M,
                                float* h, void* stream) {
  clear_error();
  if (int rc = lora_args("lora_shrink", dtype, r, L, M, K)) return rc;
  if (M == 0) return MXGG_OK;
  if (!x || !w || !src || !offs || !h) return fail(MXGG_ERR_INVALID_ARG, "lora_shrink: null pointer");
  if (ldx < 0 || (ldw_r < K && r > 1) || ldw_l < 0) return fail(MXGG_ERR_INVALID_ARG, "lora_shrink: row stride below K=%lld", (long long)K);
  if (int rc = require_device()) return rc;
  const int S = shrink_splits(M, L, r, K);
  hipStream_t st = (hipStream_t)stream;
  return dtype == MXGG_DTYPE_BF16 ? launch_shrink<__bf16>(x, ldx, K, w, ldw_r, ldw_l, r, src, offs, L, M, h, S, st)
                                  : launch_shrink<_Float16>(x, ldx, K, w, ldw_r, ldw_l, r, src, offs, L, M, h, S, st);
}

extern "C" int mxgg_lora_expand(const float* h, int64_t h_floats, const void* w, int dtype, int64_t N, int64_t ldw_r,
                                int64_t ldw_l, int r, const float* scales, const void* base, int64_t ldb, void* out,
                                int64_t ldo, const int32_t* rows, int64_t tokens, const int32_t* src,
                                const int32_t* offs, int L, int64_t M, void* stream) {
  clear_error();
  if (int rc = lora_args("lora_expand", dtype, r, L, M, N)) return rc;
  if (tokens == 0) return MXGG_OK;
  if (M == 0 || h_floats < M * rank_pad(r) || h_floats % (M * rank_pad(r)))
    return fail(MXGG_ERR_INVALID_ARG, "lora_expand: %lld floats do not hold %lld rows", (long long)h_floats, (long long)M);
  if (!h || !w || !out || !rows || !src || !offs) return fail(MXGG_ERR_INVALID_ARG, "lora_expand: null pointer");
  if ((ldw_r < N && r > 1) || (tokens > 1 && (ldo < N || (base && ldb < N))))
    return fail(MXGG_ERR_INVALID_ARG, "lora_expand: row stride below N=%lld", (long long)N);
  if (int rc = require_device()) return rc;
  const int S = (int)(h_floats / (M * rank_pad(r)));
  hipStream_t st = (hipStream_t)stream;
  return dtype == MXGG_DTYPE_BF16
             ? launch_expand<__bf16>(h, S, M, w, ldw_r, ldw_l, r, N, scales, base, ldb, out, ldo, rows, tokens, src, offs, L, st)
             : launch_expand<_Float16>(h, S, M, w, ldw_r, ldw_l, r, N, scales, base, ldb, out, ldo, rows, tokens, src, offs, L, st);
}

extern "C" int mxgg_lora_outer(const float* h, int64_t h_floats, const void* x, int dtype, int64_t K, int64_t ldx, int r,
                               const float* scales, const int32_t* src, const int32_t* offs, int L, int64_t M,
                               void* out, float* workspace, int64_t ws_floats, void* stream) {
  clear_error();
  if (int rc = lora_args("lora_outer", dtype, r, L, M, K)) return rc;
  if (M == 0 || h_floats < M * rank_pad(r) || h_floats % (M * rank_pad(r)))
    return fail(MXGG_ERR_INVALID_ARG, "lora_outer: %lld floats do not hold %lld rows", (long long)h_floats, (long long)M);
  if (!h || !x || !src || !offs || !out) return fail(MXGG_ERR_INVALID_ARG, "lora_outer: null pointer");
  if (ldx < 0) return fail(MXGG_ERR_INVALID_ARG, "lora_outer: negative row stride");
  const int64_t need = mxgg_lora_outer_floats(M, L, r, K);
  if (need && (!workspace || ws_floats < need))
    return fail(MXGG_ERR_WORKSPACE, "lora_outer: workspace of %lld floats needed", (long long)need);
  if (int rc = require_device()) return rc;
  const int S = (int)(h_floats / (M * rank_pad(r)));
  hipStream_t st = (hipStream_t)stream;
  return dtype == MXGG_DTYPE_BF16
             ? launch_outer<__bf16>(h, S, M, r, x, ldx, K, scales, src, offs, L, out, workspace, st)
             : launch_outer<_Float16>(h, S, M, r, x, ldx, K, scales, src, offs, L, out, workspace, st);
}
