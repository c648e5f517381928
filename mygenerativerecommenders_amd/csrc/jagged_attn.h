// Shared pieces of the per-head softmax attention over jagged rows (forward and backward).
//
// All products run on the matrix cores with 32 x 32 accumulator tiles: bf16 operands
// (16 contraction steps an instruction) or fp32 operands (2 steps), fp32 accumulation.
// A wave computes its score tiles transposed to what its next product contracts, so a
// tile of probabilities goes from the accumulators of one product into the operand of the
// next without leaving the registers: accumulator register r of lane half h holds row
// (r & 3) + 8 (r >> 2) + 4 h, and the other operand is read from LDS in that row order.
#pragma once

#include "common.h"
#include "mfma32.h"

namespace gr {

struct JaggedAttnArgs {
  const void* q;
  int64_t ld_q, hs_q;  // element strides of a row and of a head
  const void* k;
  int64_t ld_k, hs_k;
  const void* v;
  int64_t ld_v, hs_v;
  const int64_t* offsets;
  int B;
  int64_t rows;
  int Hkv, group;  // query heads = Hkv * group
  int d, dv;
  int causal;
  float scale;     // of the scores
  float scale_l2;  // scale / ln 2
  void* out;       // (rows, H, dv)
  float* lse;      // (H, rows): log2 of each row's sum of 2^(scaled score / ln 2), or NULL
  const void* dout;  // (rows, H, dv)
  void* dq;          // (rows, H, d)
  void* dk;          // (rows, Hkv, d)
  void* dvv;         // (rows, Hkv, dv)
  float* delta;      // (H, rows): sum(dout * out)
  int64_t slots;     // tiles of the rows per head, see jagged_tile
};

// Tile `slot` of the jagged rows in tiles of BM rows that never cross a sequence: sequence b
// owns the slots from offsets[b] / BM + b on, which always leaves it enough of them, so
// neither the longest length nor a prefix of tile counts is needed on the host.  The rows
// past the last sequence are tiled as one more (`tail`).  A search over the offsets, 64 at a
// time.  Offsets outside the rows are clamped.
struct JaggedTile {
  int64_t s0;  // first row of the sequence
  int len;     // its length (0: the slot holds no tile)
  int r0;      // first row of the tile in the sequence
  bool tail;   // rows of no sequence
};
inline int64_t jagged_slots(int64_t rows, int B, int bm) { return rows / bm + B + 1; }
__device__ __forceinline__ int64_t ja_clamp(int64_t x, int64_t lo, int64_t hi) { return x < lo ? lo : x > hi ? hi : x; }
template <int BM>
__device__ __forceinline__ JaggedTile jagged_tile(const int64_t* offsets, int B, int64_t rows, int64_t slot) {
  int lo = 0, hi = B + 1;
  const int lane = threadIdx.x & 63;
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) >> 6;
    const int i = lo + lane * step;
    const bool le = i < hi && ja_clamp(offsets[i < hi ? i : B], 0, rows) / BM + i <= slot;
    const int c = __popcll(__ballot(le));
    lo += (c > 0 ? c - 1 : 0) * step;
    hi = hi < lo + step ? hi : lo + step;
  }
  JaggedTile t;
  t.s0 = ja_clamp(offsets[lo], 0, rows);
  t.tail = lo == B;
  const int64_t end = t.tail ? rows : ja_clamp(offsets[lo + 1], t.s0, rows);
  const int64_t r0 = (slot - lo - t.s0 / BM) * BM;
  t.len = r0 >= 0 && r0 < end - t.s0 ? (int)(end - t.s0) : 0;
  t.r0 = (int)r0;
  return t;
}

// 16 bytes of a row from column c, for rows of `d` elements of any alignment, in two steps so
// that the first can stay in flight: ja_load16 reads inside the row always (the vector that
// would cross its end is read up against it), ja_fix16 moves such a vector's elements down
// and clears what lies past column d, or all of it where `ok` is false.
template <typename T>
__device__ __forceinline__ u32x4_t ja_load16(const T* row, int c, int d) {
  constexpr int V = 16 / sizeof(T);
  struct __attribute__((packed, aligned(sizeof(T)))) P {
    u32x4_t v;
  };
  if (d >= V) return reinterpret_cast<const P*>(row + min(c, d - V))->v;  // uniform
  T x[V];
#pragma unroll
  for (int i = 0; i < V; ++i) x[i] = row[min(i, d - 1)];
  u32x4_t r;
  __builtin_memcpy(&r, x, 16);
  return r;
}
template <typename T>
__device__ __forceinline__ u32x4_t ja_fix16(u32x4_t x, int c, int d, bool ok) {
  constexpr int V = 16 / sizeof(T);
  if (d % V != 0) {  // uniform
    unsigned __int128 w = __builtin_bit_cast(unsigned __int128, x);
    if (d > V)
      w >>= max(c + V - d, 0) * 8 * (int)sizeof(T) & 127;  // c >= d is cleared below
    else
      w &= ~(unsigned __int128)0 >> (V - d) * 8 * (int)sizeof(T);
    x = __builtin_bit_cast(u32x4_t, w);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = ok && c < d ? x[i] : 0u;
  return x;
}

// R rows of DP columns of a jagged operand, through the registers into LDS (256 threads).
template <typename T, int DP, int R>
struct JaStage {
  static constexpr int V = 16 / sizeof(T), CPR = DP / V, PER = R * CPR / 256;
  static_assert(R * CPR % 256 == 0, "whole passes");
  u32x4_t x[PER];
  __device__ __forceinline__ void load(const T* base, int64_t ld, int r0, int len, int d) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int at = threadIdx.x + 256 * i;
      x[i] = ja_load16<T>(base + (int64_t)min(r0 + at / CPR, len - 1) * ld, at % CPR * V, d);
    }
  }
  __device__ __forceinline__ void store(T* lds, int stride, int r0, int len, int d) {
    if (r0 + R > len || d != DP) {  // uniform
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int at = threadIdx.x + 256 * i;
        x[i] = ja_fix16<T>(x[i], at % CPR * V, d, r0 + at / CPR < len);
      }
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int at = threadIdx.x + 256 * i;
      *reinterpret_cast<u32x4_t*>(lds + at / CPR * stride + at % CPR * V) = x[i];
    }
  }
};

// Operand fragments.  `K` contraction steps of a fragment: 16 (bf16) or 8 (fp32); lane half
// h holds the 16 bytes of columns K s + (K / 2) h on of row lane % 32.
template <typename T>
struct JaFrag;
template <>
struct JaFrag<__bf16> {
  static constexpr int K = 16;
  static __device__ __forceinline__ f32x16 mma(u32x4_t a, u32x4_t b, f32x16 c) { return mfma32(a, b, c); }
  // A product that contracts 32 rows held in accumulators `p`: c += X^T p with X the LDS
  // rows of a tile, columns c0 .. c0 + 31.  `p` is rounded to bf16 (half a step: 2^-9 of each
  // probability, as its bf16 neighbours in the product).
  struct Rows {
    u32x4_t x[2];
    __device__ __forceinline__ explicit Rows(const f32x16& p) {
#pragma unroll
      for (int s = 0; s < 2; ++s)
        x[s] = u32x4_t{pack_bf16(p[8 * s], p[8 * s + 1]), pack_bf16(p[8 * s + 2], p[8 * s + 3]),
                       pack_bf16(p[8 * s + 4], p[8 * s + 5]), pack_bf16(p[8 * s + 6], p[8 * s + 7])};
    }
    __device__ __forceinline__ f32x16 mma(const __bf16* tile, int stride, int c0, f32x16 c) const {
      const int lane = threadIdx.x & 63;
#pragma unroll
      for (int s = 0; s < 2; ++s) c = mfma32(trB_acc(tile, stride, s, c0, lane), x[s], c);
      return c;
    }
  };
};
template <>
struct JaFrag<float> {
  static constexpr int K = 8;
  static __device__ __forceinline__ f32x16 mma1(float a, float b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16 mma(u32x4_t a, u32x4_t b, f32x16 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = mma1(__uint_as_float(a[i]), __uint_as_float(b[i]), c);
    return c;
  }
  struct Rows {
    const f32x16& x;
    __device__ __forceinline__ explicit Rows(const f32x16& p) : x(p) {}
    __device__ __forceinline__ f32x16 mma(const float* tile, int stride, int c0, f32x16 c) const {
      const int lane = threadIdx.x & 63, h = lane >> 5;
      const float* at = tile + 4 * h * stride + c0 + (lane & 31);
#pragma unroll
      for (int r = 0; r < 16; ++r) c = mma1(at[((r & 3) + 8 * (r >> 2)) * stride], x[r], c);
      return c;
    }
  };
};

// A wave's 32 rows of an operand as fragments: in registers, or (where the registers of the
// widest fp32 heads do not hold them) read again from cache at every use.
template <typename T, int DP, bool KEEP>
struct JaRows {
  static constexpr int K = JaFrag<T>::K, KS = DP / K;
  u32x4_t x[KEEP ? KS : 1];
  const T* row;
  int d;
  bool ok;
  __device__ __forceinline__ void init(const T* base, int64_t ld, int r0, int len, int width) {
    const int lane = threadIdx.x & 63, r = r0 + (lane & 31);
    ok = r < len;
    row = base + (int64_t)min(r, len - 1) * ld;
    d = width;
    if constexpr (KEEP) {
#pragma unroll
      for (int s = 0; s < KS; ++s) x[s] = ja_load16<T>(row, col(s), d);
#pragma unroll
      for (int s = 0; s < KS; ++s) x[s] = ja_fix16<T>(x[s], col(s), d, ok);
    }
  }
  static __device__ __forceinline__ int col(int s) { return K * s + K / 2 * ((threadIdx.x & 63) >> 5); }
  // Keeps what follows from being read before it (and held in registers after all).
  __device__ __forceinline__ void renew() {
    if constexpr (!KEEP) asm volatile("" : "+v"(row));
  }
  __device__ __forceinline__ u32x4_t at(int s) const {
    if constexpr (KEEP) return x[s];
    return ja_fix16<T>(ja_load16<T>(row, col(s), d), col(s), d, ok);
  }
};

// c = X Y^T over 32 x 32: X rows from LDS (row-major tile), Y the wave's fragments.
template <typename T, int DP, bool KEEP>
__device__ __forceinline__ f32x16 ja_scores(const T* tile, int stride, JaRows<T, DP, KEEP>& y) {
  using F = JaFrag<T>;
  const int lane = threadIdx.x & 63;
  const T* row = tile + (lane & 31) * stride + F::K / 2 * (lane >> 5);
  f32x16 c = f16_zero();
#pragma unroll
  for (int s = 0; s < DP / F::K; ++s) {
    if (s % 8 == 0) y.renew();
    c = F::mma(*reinterpret_cast<const u32x4_t*>(row + F::K * s), y.at(s), c);
  }
  return c;
}

// Accumulators of a transposed result (register = column of the row lane % 32) to memory.
template <typename T>
__device__ __forceinline__ void ja_store_t(T* row, int c0, int width, const f32x16& v, float f, bool ok) {
  const int h = (threadIdx.x & 63) >> 5;
  if (!ok) return;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int c = c0 + 8 * g + 4 * h;
    if (c + 4 <= width) {
      struct __attribute__((packed, aligned(sizeof(T)))) P {
        T v[4];
      };
      P p;
#pragma unroll
      for (int i = 0; i < 4; ++i) p.v[i] = (T)(v[4 * g + i] * f);
      *reinterpret_cast<P*>(row + c) = p;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (c + i < width) row[c + i] = (T)(v[4 * g + i] * f);
    }
  }
}

// Zeros in `width` columns of n rows.
template <typename T>
__device__ __forceinline__ void ja_zero(T* base, int64_t ld, int n, int width) {
  for (int i = threadIdx.x; i < n * width; i += 256) base[(int64_t)(i / width) * ld + i % width] = (T)0.f;
}

__device__ __forceinline__ float swap_half(float v) { return __shfl_xor(v, 32, 64); }

// LDS row strides (elements).  Read by rows (16 bytes a lane) a stride of an odd number of
// 16-byte units spreads the banks; read transposed, 4 or 8 rows at once, one of 64 bytes
// beyond a multiple of 128 does.
template <typename T>
__host__ __device__ constexpr int ja_row_stride(int dp) { return dp + 16 / (int)sizeof(T); }
template <typename T>
__host__ __device__ constexpr int ja_col_stride(int dp) { return dp + (sizeof(T) == 2 ? 32 : 8); }

// Whether a wave's 32 rows of an operand (and the accumulators beside them) fit its registers.
template <typename T, int DP>
constexpr bool ja_keep = sizeof(T) == 2 || DP <= 128;

int jagged_attn_check(const char* what, const JaggedAttnArgs& a, int H);

}  // namespace gr
