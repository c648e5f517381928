// Shared pieces of the per-head softmax attention over jagged rows (forward and backward).
//
// All products run on the matrix cores with 32 x 32 accumulator tiles: bf16 operands
// (16 contraction steps an instruction) or fp32 operands (2 steps), fp32 accumulation.
// A wave computes its score tiles transposed to what its next product contracts, so a
// tile of probabilities goes from the accumulators of one product into the operand of the
// next without leaving the registers: accumulator register r of lane half h holds row
// (r & 3) + 8 (r >> 2) + 4 h, and the other operand is read from LDS in that row order.
#pragma once

#include <type_traits>

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
  void* out_low;   // bf16: what out's rounding left off, or NULL
  float* lse;      // (H, rows): log2 of each row's sum of 2^(scaled score / ln 2), +inf from 2^23 on, or NULL
  const void* dout;  // (rows, H, dv)
  void* dq;          // (rows, H, d)
  void* dk;          // (rows, Hkv, d)
  void* dvv;         // (rows, Hkv, dv)
  float* delta;      // (H, rows): sum(dout * out)
  int64_t slots;     // tiles of the rows per head, see jagged_tile
  int wide;          // rows and their starts are multiples of 16 bytes
};

// Work item of a workgroup: slot, key head, and query head of its group.  Workgroups i, i + 8, ..
// land on one XCD: the heads of a group follow each other there, so that its L2 serves them the
// same keys and values.
struct JaggedWork {
  int hk, g;
  int64_t slot;  // >= slots: nothing
};
inline int64_t jagged_grid(int64_t slots, int Hkv, int group) { return (slots * Hkv + 7) / 8 * 8 * group; }
__device__ __forceinline__ JaggedWork jagged_work(const JaggedAttnArgs& a, unsigned group, unsigned id) {
  const unsigned j = id / 8, u = j / group * 8 + id % 8;
  JaggedWork k;
  k.g = (int)(j % group);
  k.slot = u / (unsigned)a.Hkv;
  k.hk = (int)(u % (unsigned)a.Hkv);
  return k;
}

// Sum over the wave, in every lane.
__device__ __forceinline__ int wave_isum(int v) {
  auto mov = [](int x, auto ctrl) { return __builtin_amdgcn_update_dpp(0, x, decltype(ctrl)::value, 0xF, 0xF, true); };
  v += mov(v, std::integral_constant<int, 0xB1>{});   // quad_perm [1,0,3,2]
  v += mov(v, std::integral_constant<int, 0x4E>{});   // quad_perm [2,3,0,1]
  v += mov(v, std::integral_constant<int, 0x141>{});  // row_half_mirror
  v += mov(v, std::integral_constant<int, 0x140>{});  // row_mirror
  return __builtin_amdgcn_readlane(v, 0) + __builtin_amdgcn_readlane(v, 16) + __builtin_amdgcn_readlane(v, 32) +
         __builtin_amdgcn_readlane(v, 48);
}

// Maximum over the wave, in every lane; values >= 0.
__device__ __forceinline__ int wave_imax(int v) {
  auto mov = [](int x, auto ctrl) { return __builtin_amdgcn_update_dpp(0, x, decltype(ctrl)::value, 0xF, 0xF, true); };
  v = max(v, mov(v, std::integral_constant<int, 0xB1>{}));
  v = max(v, mov(v, std::integral_constant<int, 0x4E>{}));
  v = max(v, mov(v, std::integral_constant<int, 0x141>{}));
  v = max(v, mov(v, std::integral_constant<int, 0x140>{}));
  return max(max(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16)),
             max(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48)));
}

// Tile `slot` of the jagged rows in tiles of BM rows that never cross a sequence; the rows before
// the first and past the last sequence are tiled as one more each (`none`).  The host knows neither
// lengths nor tile counts, only that rows / BM + B + 2 slots are enough.  Offsets are clamped to
// the rows.
//
// Up to 255 sequences the wave holds them all, and slots run from the heavy tiles to the light
// ones: level n of a sequence is the tile that meets n tiles of a causal sequence's other side
// (`keys`: the key rows' pass, where that is the n-th from the end), slots go down the levels
// and through the sequences that reach them.  Workgroups start in that order, so the longest
// do not run alone at the end.  With more sequences, sequence b owns the slots from
// offsets[b] / BM + b + 1 on, found by a search over the offsets, 64 at a time.
struct JaggedTile {
  int64_t s0;  // first row of the sequence
  int len;     // its length (0: the slot holds no tile)
  int r0;      // first row of the tile in the sequence
  bool none;   // rows of no sequence
};
inline int64_t jagged_slots(int64_t rows, int B, int bm) { return rows / bm + B + 2; }
__device__ __forceinline__ int64_t ja_clamp(int64_t x, int64_t lo, int64_t hi) { return x < lo ? lo : x > hi ? hi : x; }
template <int BM, bool KEYS>
__device__ __forceinline__ JaggedTile jagged_tile(const int64_t* offsets, int B, int64_t rows, int64_t slot) {
  const int lane = threadIdx.x & 63;
  JaggedTile t;
  t.none = false;
  if (B < 256) {
    int first[4], tiles[4], lens[4], total = 0;  // rows < 2^31
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      first[j] = tiles[j] = lens[j] = 0;
      if (64 * j < B) {  // uniform
        const int i = 64 * j + lane;
        const int64_t lo = ja_clamp(offsets[i < B ? i : B], 0, rows), hi = ja_clamp(offsets[i < B ? i + 1 : B], lo, rows);
        first[j] = (int)lo;
        lens[j] = i < B ? (int)(hi - lo) : 0;
        tiles[j] = (lens[j] + BM - 1) / BM;
      }
    }
    auto above = [&](int n) {  // tiles of level n and more
      int c = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) c += tiles[j] >= n ? tiles[j] - n + 1 : 0;
      return wave_isum(c);
    };
    total = above(1);
    if (slot >= total) {
      const int64_t start = ja_clamp(B > 0 ? offsets[0] : 0, 0, rows), end = ja_clamp(B > 0 ? offsets[B] : 0, start, rows);
      const int64_t before = (start + BM - 1) / BM, i = slot - total;
      const bool head = i < before;
      const int64_t r0 = (head ? i : i - before) * BM, n = head ? start : rows - end;
      t.none = true;
      t.s0 = head ? 0 : end;
      t.len = r0 < n ? (int)n : 0;
      t.r0 = (int)r0;
      return t;
    }
    // level n has the slot or is below it, level `more` is empty or above it
    int n = 1, more = wave_imax(max(max(tiles[0], tiles[1]), max(tiles[2], tiles[3]))) + 1, past = 0;
    while (more - n > 1) {
      const int mid = (n + more) >> 1, c = above(mid);
      if (c > slot) {
        n = mid;
      } else {
        more = mid;
        past = c;
      }
    }
    int k = (int)slot - past;  // the k-th sequence that reaches level n
    t.s0 = 0;
    t.len = t.r0 = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const unsigned long long reach = __ballot(tiles[j] >= n);
      const int c = __popcll(reach);
      if (k >= 0 && k < c) {  // uniform
        const bool me = tiles[j] >= n && (int)__popcll(reach & ((1ull << lane) - 1ull)) == k;
        const int at = __ffsll(__ballot(me)) - 1;
        t.s0 = __builtin_amdgcn_readlane(first[j], at);
        t.len = __builtin_amdgcn_readlane(lens[j], at);
        t.r0 = (KEYS ? __builtin_amdgcn_readlane(tiles[j], at) - n : n - 1) * BM;
      }
      k = k < c ? -1 : k - c;
    }
    return t;
  }
  auto start = [&](int i) { return i > 0 ? ja_clamp(offsets[i - 1], 0, rows) : 0; };  // of sequence i - 1
  int lo = 0, hi = B + 2;
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) >> 6;
    const int i = lo + lane * step;
    const bool le = i < hi && start(i < hi ? i : 0) / BM + i <= slot;
    const int c = __popcll(__ballot(le));
    lo += (c > 0 ? c - 1 : 0) * step;
    hi = hi < lo + step ? hi : lo + step;
  }
  t.s0 = start(lo);
  t.none = lo == 0 || lo == B + 1;
  const int64_t end = lo == B + 1 ? rows : ja_clamp(offsets[lo], t.s0, rows);
  const int64_t r0 = (slot - lo - t.s0 / BM) * BM;
  t.len = r0 >= 0 && r0 < end - t.s0 ? (int)(end - t.s0) : 0;
  t.r0 = (int)r0;
  return t;
}

// 16 bytes of a row from column c, for rows of `d` >= 16 bytes of any alignment, in two steps
// so that the first can stay in flight: ja_load16 reads inside the row always (the vector
// that would cross its end is read up against it), ja_fix16 moves such a vector's elements
// down and clears what lies past column d.
template <typename T>
__device__ __forceinline__ u32x4_t ja_load16(const T* row, int c, int d) {
  constexpr int V = 16 / sizeof(T);
  struct __attribute__((packed, aligned(sizeof(T)))) P {
    u32x4_t v;
  };
  return reinterpret_cast<const P*>(row + min(c, d - V))->v;
}
template <typename T>
__device__ __forceinline__ u32x4_t ja_fix16(u32x4_t x, int c, int d) {
  constexpr int V = 16 / sizeof(T);
  if (d % V != 0) {  // uniform
    unsigned __int128 w = __builtin_bit_cast(unsigned __int128, x);
    w >>= max(c + V - d, 0) * 8 * (int)sizeof(T) & 127;  // c >= d is cleared below
    x = __builtin_bit_cast(u32x4_t, w);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = c < d ? x[i] : 0u;
  return x;
}

// LDS tiles: R rows of DP columns in 16-byte units, 64 of them (RPI rows, 1 KB: what one
// load-to-LDS instruction writes) followed by one of padding; unit c of row r at place
// c ^ swizzle(r) of its row.  Read by rows (each lane a row, the same unit) 16 rows cover the 64
// banks once; read transposed (4 neighbouring units of 8 rows) no bank is hit more often than
// the bytes take.  Swizzles change few bits, so that most of an address is a constant.
template <typename T, int DP>
struct JaTile {
  static constexpr int V = 16 / sizeof(T), UNITS = DP / V, RPI = 64 / UNITS;
  static constexpr int BITS = RPI == 8 ? 6 : RPI == 4 ? 12 : RPI == 2 ? 8 : 0;  // that a swizzle changes
  static __host__ __device__ constexpr int size(int rows) { return rows / RPI * 65; }
  static __device__ __forceinline__ int swizzle(int r) {
    return RPI == 8 ? (r >> 1 & 3) << 1 : RPI == 4 ? (r & 3) << 2 : RPI == 2 ? (r & 1) << 3 : 0;
  }
  // Unit c0 + cl of row r0 + r: r0 a multiple of 8, c0 of LOW > cl; r0 and c0 constants.
  template <int LOW>
  static __device__ __forceinline__ int unit(int r0, int r, int c0, int cl) {
    const int f = swizzle(r);
    return r / RPI * 65 + r % RPI * UNITS + (cl ^ (f & (LOW - 1))) + ((c0 & BITS) ^ (f & ~(LOW - 1))) +
           (c0 & ~BITS) + size(r0);
  }
};
// Brings R rows of a jagged operand into an LDS tile, with a set of QW waves, straight from
// memory (buffer loads to LDS of BYTES a lane: 16 where rows and their starts are multiples of
// that, else 4).  They are issued where the compiler does not see them, so that it does not
// wait for them at the next LDS read: ja_landed() waits and meets the other waves.  The
// descriptor ends with the sequence's last row, so rows past it come as zeros where the stride is
// d or more (below, as rows of the sequence: only callers that mask by index take such), and lanes
// past column d ask for what is out of its range.
template <typename T, int DP, int R, int BYTES, int QW>
struct JaStage {
  using Tile = JaTile<T, DP>;
  static constexpr int SZ = sizeof(T), PER = 16 / BYTES;             // lanes that share a unit
  static constexpr int N = R * Tile::UNITS * PER / (64 * QW);        // instructions of a wave
  // an instruction writes 1 / PER of a kilobyte of the tile; the waves take them in turn, so a
  // wave meets PH different parts of a kilobyte, each with its own columns
  static constexpr int PH = PER > QW ? PER / QW : 1, BLOCKS = QW > PER ? QW / PER : 1;  // kilobytes a turn
  static_assert(R * Tile::UNITS * PER % (64 * QW) == 0 && Tile::UNITS <= 64, "whole instructions");
  uint32_t off[PH], at;  // this wave's place in memory and in the tile at LDS address 0
  uint64_t p;            // the next tile's first row
  int64_t left;          // bytes from there to the end of the sequence's last row
  int row;               // of a row
  // Rows r0 on of a sequence's `len`, d columns wide.
  __device__ __forceinline__ void init(const T* base, int64_t ld, int r0, int len, int d) {
    const int lane = threadIdx.x & 63, w = wave_id() % QW;
    row = (int)ld * SZ;  // ld < 2^22
#pragma unroll
    for (int i = 0; i < PH; ++i) {
      const int u = (i * QW + w) * 64 / PER + lane / PER, r = u / Tile::UNITS;
      const int c = (u % Tile::UNITS ^ Tile::swizzle(r)) * Tile::V + lane % PER * (BYTES / SZ);
      off[i] = c < d ? (uint32_t)(r * row + c * SZ) : (uint32_t)OOB_OFF;
    }
    at = 1040u * (w / PER) + 1024u / PER * (w % PER);
    seek(base, r0, len, d);
  }
  __device__ __forceinline__ void seek(const T* base, int r0, int len, int d) {
    p = (uint64_t)base + (int64_t)r0 * row;
    left = (int64_t)(len - r0 - 1) * row + d * SZ;
  }
  // The tile at p to LDS, and p on by `rows`.
  __device__ __forceinline__ void load(uint32_t lds, int rows) {
    const u32x4_t desc = {(uint32_t)p, (uint32_t)(p >> 32) & 0xFFFFu, (uint32_t)(left < 0x7FFFFFFF ? left : 0x7FFFFFFF),
                          0x00020000u};
    const uint32_t base = __builtin_amdgcn_readfirstlane(lds + at);
    auto to = [&](int i) { return base + 1040u * BLOCKS * (i / PH) + (i % PH) * (1024u / PER * QW); };
    int turn = BLOCKS * Tile::RPI * row;
    asm volatile("" : "+s"(turn));  // its multiples are made here, not kept in registers
    auto from = [&](int i) { return i / PH * turn; };
    uint32_t keep;  // m0 is saved and put back: the compiler may hold something in it
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      if constexpr (N % 2 != 0) {
        static_assert(N == 1 && BYTES == 16);
        asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, %4 offen lds\n\t"
                     "s_mov_b32 m0, %0"
                     : "=&s"(keep) : "s"(to(i)), "v"(off[0]), "s"(desc), "s"(from(i)) : "memory");
      } else if constexpr (BYTES == 16) {
        asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, %4 offen lds\n\t"
                     "s_mov_b32 m0, %5\n\ts_nop 0\n\tbuffer_load_dwordx4 %6, %3, %7 offen lds\n\ts_mov_b32 m0, %0"
                     : "=&s"(keep)
                     : "s"(to(i)), "v"(off[i % PH]), "s"(desc), "s"(from(i)), "s"(to(i + 1)), "v"(off[(i + 1) % PH]),
                       "s"(from(i + 1))
                     : "memory");
      } else {
        asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tbuffer_load_dword %2, %3, %4 offen lds\n\t"
                     "s_mov_b32 m0, %5\n\ts_nop 0\n\tbuffer_load_dword %6, %3, %7 offen lds\n\ts_mov_b32 m0, %0"
                     : "=&s"(keep)
                     : "s"(to(i)), "v"(off[i % PH]), "s"(desc), "s"(from(i)), "s"(to(i + 1)), "v"(off[(i + 1) % PH]),
                       "s"(from(i + 1))
                     : "memory");
      }
    }
    p += (int64_t)rows * row;
    left -= (int64_t)rows * row;
  }
};
template <typename V>
__device__ __forceinline__ uint32_t ja_lds(const V* at) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const V*)at;
}
// The same for one float a lane (lanes < N of a wave): p[0 .. left - 1], zeros past them.
template <int N>
__device__ __forceinline__ void ja_stage_floats(const float* p, int left, uint32_t lds) {
  const uint64_t at = (uint64_t)p;
  const u32x4_t desc = {(uint32_t)at, (uint32_t)(at >> 32) & 0xFFFFu, (uint32_t)min(left, N) * 4u, 0x00020000u};
  const uint32_t base = __builtin_amdgcn_readfirstlane(lds);
  const int lane = threadIdx.x & 63;
  uint32_t keep;
  if (N == 64 || lane < N)
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tbuffer_load_dword %2, %3, 0 offen lds\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "s"(base), "v"(4 * lane), "s"(desc) : "memory");
}
__device__ __forceinline__ void ja_landed() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Operand fragments.  `K` contraction steps of a fragment: 16 (bf16) or 8 (fp32); lane half
// h holds the 16 bytes of columns K s + (K / 2) h on of row lane % 32.
template <typename T>
struct JaFrag;
template <>
struct JaFrag<__bf16> {
  static constexpr int K = 16;
  static __device__ __forceinline__ f32x16 mma(u32x4_t a, u32x4_t b, f32x16 c) { return mfma32(a, b, c); }
  // A product that contracts 32 rows held in accumulators `p`: c += X^T p with X rows r0 ..
  // r0 + 31 of a tile, columns 32 t .. 32 t + 31.  `p` is rounded to bf16 (half a step: 2^-8 of
  // each value), as its neighbours in the product are bf16.
  struct Rows {
    u32x4_t x[2];
    __device__ __forceinline__ explicit Rows(const f32x16& p) {
#pragma unroll
      for (int s = 0; s < 2; ++s)
        x[s] = u32x4_t{pack_bf16(p[8 * s], p[8 * s + 1]), pack_bf16(p[8 * s + 2], p[8 * s + 3]),
                       pack_bf16(p[8 * s + 4], p[8 * s + 5]), pack_bf16(p[8 * s + 6], p[8 * s + 7])};
    }
    // What the rounding of `p` left off.
    __device__ __forceinline__ Rows low(const f32x16& p) const {
      f32x16 e;
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          e[8 * s + 2 * i] = p[8 * s + 2 * i] - __uint_as_float(x[s][i] << 16);
          e[8 * s + 2 * i + 1] = p[8 * s + 2 * i + 1] - __uint_as_float(x[s][i] & 0xFFFF0000u);
        }
      return Rows(e);
    }
    // Transposed reads: lane 4 q + p of a 16-lane group addresses row q, columns 4 p on of a
    // 4 x 16 block and receives column lane % 16 of its 4 rows.
    template <int DP, bool LOW = false>
    __device__ __forceinline__ f32x16 mma(const u32x4_t* tile, int r0, int t, f32x16 c, const Rows* e = nullptr) const {
      using Tile = JaTile<__bf16, DP>;
      const int lane = threadIdx.x & 63, g = lane >> 4, q = (lane & 15) >> 2, p = lane & 3;
      const int row = 4 * (lane >> 5) + q, cl = 2 * (g & 1) + (p >> 1);
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const u32x4_t *lo = tile + Tile::template unit<4>(r0 + 16 * s, row, 4 * t, cl), *hi = lo + Tile::size(8);
        const u32x2_t a = tr16(reinterpret_cast<const __bf16*>(lo) + 4 * (p & 1)),
                      b = tr16(reinterpret_cast<const __bf16*>(hi) + 4 * (p & 1));
        c = mfma32(u32x4_t{a.x, a.y, b.x, b.y}, x[s], c);
        if constexpr (LOW) c = mfma32(u32x4_t{a.x, a.y, b.x, b.y}, e->x[s], c);
      }
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
    template <int DP>
    __device__ __forceinline__ f32x16 mma(const u32x4_t* tile, int r0, int t, f32x16 c) const {
      using Tile = JaTile<float, DP>;
      const int lane = threadIdx.x & 63, h = lane >> 5;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float* at = reinterpret_cast<const float*>(
            tile + Tile::size(4) * h + Tile::template unit<8>(r0 + 8 * (r >> 2), r & 3, 8 * t, (lane & 31) / 4));
        c = mma1(at[lane & 3], x[r], c);
      }
      return c;
    }
  };
};

// A wave's 32 rows of an operand as fragments: in registers, or (where the registers of the
// widest fp32 heads do not hold them) read again from cache at every use.  Rows past the end
// repeat the last one: what comes of them is not stored.
template <typename T, int DP, bool KEEP>
struct JaRows {
  static constexpr int K = JaFrag<T>::K, KS = DP / K;
  u32x4_t x[KEEP ? KS : 1];
  const T* row;
  int d;
  __device__ __forceinline__ void init(const T* base, int64_t ld, int r0, int len, int width) {
    const int lane = threadIdx.x & 63, r = r0 + (lane & 31);
    row = base + (int64_t)min(r, len - 1) * ld;
    d = width;
    if constexpr (KEEP) {
#pragma unroll
      for (int s = 0; s < KS; ++s) x[s] = ja_load16<T>(row, col(s), d);
#pragma unroll
      for (int s = 0; s < KS; ++s)
        if (K * s + K > d) x[s] = ja_fix16<T>(x[s], col(s), d);
    }
  }
  static __device__ __forceinline__ int col(int s) { return K * s + K / 2 * ((threadIdx.x & 63) >> 5); }
  // Keeps what follows from being read before it (and held in registers after all).
  __device__ __forceinline__ void renew() {
    if constexpr (!KEEP) asm volatile("" : "+v"(row));
  }
  __device__ __forceinline__ u32x4_t at(int s) const {
    if constexpr (KEEP) return x[s];
    const u32x4_t v = ja_load16<T>(row, col(s), d);
    return K * s + K > d ? ja_fix16<T>(v, col(s), d) : v;
  }
};

// c = X Y^T over 32 x 32: X rows r0 .. r0 + 31 of an LDS tile, Y the wave's fragments.
template <typename T, int DP, bool KEEP>
__device__ __forceinline__ f32x16 ja_scores(const u32x4_t* tile, int r0, JaRows<T, DP, KEEP>& y) {
  using F = JaFrag<T>;
  using Tile = JaTile<T, DP>;
  const int lane = threadIdx.x & 63;
  f32x16 c = f16_zero();
#pragma unroll
  for (int s = 0; s < DP / F::K; ++s) {
    if (s % 4 == 0) y.renew();
    c = F::mma(tile[Tile::template unit<2>(r0, lane & 31, 2 * s, lane >> 5)], y.at(s), c);
  }
  return c;
}

template <typename T>
__device__ __forceinline__ void ja_floats(u32x4_t x, float (&o)[16 / sizeof(T)]) {
  T t[16 / sizeof(T)];
  __builtin_memcpy(t, &x, 16);
#pragma unroll
  for (int i = 0; i < 16 / (int)sizeof(T); ++i) o[i] = (float)t[i];
}

// Accumulators of a transposed result (register = column of the row lane % 32) to memory.
template <typename T>
__device__ __forceinline__ void ja_store_t(T* row, int c0, int width, const f32x16& v, float f, bool ok,
                                           T* low = nullptr) {
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
      if (low) {  // what the rounding left off
        P e;
#pragma unroll
        for (int i = 0; i < 4; ++i) e.v[i] = (T)(v[4 * g + i] * f - (float)p.v[i]);
        *reinterpret_cast<P*>(low + c) = e;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (c + i < width) {
          row[c + i] = (T)(v[4 * g + i] * f);
          if (low) low[c + i] = (T)(v[4 * g + i] * f - (float)row[c + i]);
        }
    }
  }
}

// Zeros in `width` columns of n rows.
template <typename T>
__device__ __forceinline__ void ja_zero(T* base, int64_t ld, int n, int width) {
  for (int i = threadIdx.x; i < n * width; i += blockDim.x) base[(int64_t)(i / width) * ld + i % width] = (T)0.f;
}

// Sets of waves that took the tiles in turn join their sums: the other sets' accumulators pass
// to the first through LDS (4 KB an accumulator and wave; the tiles' own space).
template <int QW, int DT>
__device__ __forceinline__ void ja_give(float* lds, const f32x16 (&v)[DT]) {
  float* at = lds + ((wave_id() % QW) * DT * 16) * 64 + (threadIdx.x & 63);
#pragma unroll
  for (int i = 0; i < DT; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) at[(i * 16 + r) * 64] = v[i][r];
}
template <int QW, int DT>
__device__ __forceinline__ void ja_take(const float* lds, f32x16 (&v)[DT], float mine = 1.f, float its = 1.f) {
  const float* at = lds + ((wave_id() % QW) * DT * 16) * 64 + (threadIdx.x & 63);
#pragma unroll
  for (int i = 0; i < DT; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      if (r % 8 == 0) __builtin_amdgcn_sched_barrier(0);  // few of the reads at a time: registers
      v[i][r] = v[i][r] * mine + at[(i * 16 + r) * 64] * its;
    }
}

// Maximum and sum over a lane and its counterpart in the other half of the wave.
__device__ __forceinline__ float half_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Whether a wave's 32 rows of an operand (and the accumulators beside them) fit its registers.
template <typename T, int DP>
constexpr bool ja_keep = sizeof(T) == 2 || DP <= 128;

// Whether there are at most `per_cu` tiles of 128 rows for each CU: the buffers' rows / 128 and one for
// each sequence, times heads.  (The offsets are not read on the host: spare rows count as tiles, and the
// sequences' lengths, which decide too, do not show.)  The fewer the tiles, the more wave sets share a
// workgroup's: the longest tile's time is what counts then, and with many tiles the joining is only in
// the way.  Measured over ragged batches (lengths spread evenly up to the one given), causal, us of the
// kernel, one set and more:
//   bf16, width 64, forward: 24 x 1,000 rows, 2 heads (242 tiles) 27 and 20, 32 x 2,028, 1 head (295) 48 and 34,
//   24 x 1,000, 4 heads (484) 30 and 38; dQ (width 62): 37 and 26, 67 and 44, 42 and 48; key pass: 34 and 24,
//   62 and 42, 24 x 1,499, 8 heads on 2 (338) 171 and 96;
//   width 128, forward: 2 x 8,192 rows, 4 heads (336 tiles) 234 and 182, 24 x 980, 4 heads (476) 38 and 37, 64 x
//   1,000, 2 heads (650) 42 and 52; dQ: 306 and 193, 48 and 45, 50 and 62;
//   fp32, width 64 (two sets and four), forward: 4 x 3,524 rows, 2 heads (130 tiles) 142 and 129, 128 x 211, 1 head
//   (238) 17 and 19, 24 x 980, 4 heads (476) 58 and 68; key pass: 258 and 240, 30 and 28, 106 and 116.
// Key pass at width 128: its bound lies where long sequences still gain and short ones lose, 24 x 1,000 rows,
// 4 heads (484 tiles) 61 and 42, 200 x 100, 2 heads (562) 18 and 20, 128 x 996, 8 heads on 1 (650) 405 and 284, 64 x
// 1,000, 2 heads (650) 66 and 60, 128 x 500, 2 heads (780) 44 and 50, 128 x 996, 4 heads (2,600) 200 and 224.
// At width 256 a workgroup of two sets fills a CU's LDS and one of a single set half of it, and then
// a SIMD has two waves.  Forward, 24 x 1,000 rows, 2 heads (242 tiles) 64 and 43, 32 x 2,028, 1 head (295) 117 and 81,
// 128 x 996, 4 heads (2,600) 271 and 440; dQ (width 254): 85 and 57, 155 and 110, 24 x 1,000, 4 heads (484) 95 and
// 107; key passes: 144 and 98, 272 and 177, 587 and 813.
inline bool jagged_few(const JaggedAttnArgs& a, int heads, float per_cu) {
  return (float)((a.rows / 128 + a.B) * heads) <= per_cu * device_cus();
}
// Checks the sizes and fills in the rest of the arguments.
int jagged_attn_check(const char* what, JaggedAttnArgs& a, int H, int bf16);

}  // namespace gr
