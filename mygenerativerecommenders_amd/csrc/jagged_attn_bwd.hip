// Per-head softmax attention over jagged rows, backward (gr_jagged_attn_bwd).
//
// The probabilities are recomputed from the scores and the rows' log-sums, never stored:
//   P = 2^(S scale / ln 2 - lse),  dP = dO V^T,  D = sum(dO O),  dS = P (dP - D)
//   dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO
// Two passes, each with its result in registers and no atomics, so the bits do not depend
// on the order of workgroups: one over query rows (dQ, and D for the other), one over key
// rows (dK and dV, summed over the query heads that share them).  Seven products instead
// of the five that one pass with atomic dQ sums would take (eight at widths above 128).
//
// bf16, 32 x 2,059 ragged rows, one head of 256: 259 us and 10 for D, one wave a SIMD and bound by the longest
// sequence's chain of tiles.  24 x 1,499 rows, 8 heads on 2 of 64: dQ 58, key pass 98.  128 x 996 rows, 4 heads of
// 128: 213 and 216, two waves a SIMD.  fp32 products run at an eighth of bf16's rate: 128 x 211 ragged rows, one
// head of 50: 36 us and 5 for D; a single sequence of 128 rows takes 16 and 4.
#include <math.h>

#include "jagged_attn.h"

#include "../../include/gr_hstu.h"

namespace gr {

// dQ: a workgroup per 32 QW query rows and head, a wave per 32 rows and set, tiles of BN keys.
// GIVEN: D is in `delta` already.
template <typename T, int DP, int BN, int BYTES, int QW, int SETS, bool GIVEN>
__device__ __forceinline__ void ja_dq(const JaggedAttnArgs& a, unsigned block, u32x4_t* lds) {
  using F = JaFrag<T>;
  using Tile = JaTile<T, DP>;
  constexpr int BM = 32 * QW, NB = BN / 32, DT = DP / 32, TILE = Tile::size(BN);
  static_assert(SETS * 4 * TILE * 16 >= (SETS - 1) * QW * DT * 16 * 256, "the other sets' sums fit");
  const JaggedWork wk = jagged_work(a, a.group, block);
  if (wk.slot >= a.slots) return;
  const int head = wk.hk * a.group + wk.g, H = a.Hkv * a.group;
  const JaggedTile t = jagged_tile<BM, false>(a.offsets, a.B, a.rows, wk.slot);
  if (t.len == 0) return;
  T* dq = (T*)a.dq + ((t.s0 + t.r0) * H + head) * a.d;
  if (t.none) {
    ja_zero(dq, (int64_t)H * a.d, min(BM, t.len - t.r0), a.d);
    return;
  }
  const int lane = threadIdx.x & 63, wave = wave_id(), half = lane >> 5;
  const int set = SETS > 1 ? wave / QW : 0;  // takes tiles set, set + SETS, ..
  u32x4_t *lk = lds + set * 4 * TILE, *lv = lk + 2 * TILE;
  const int q0 = t.r0 + 32 * (wave % QW), qi = q0 + (lane & 31);
  const bool ok = qi < t.len;
  const T* kb = (const T*)a.k + t.s0 * a.ld_k + wk.hk * a.hs_k;
  const T* vb = (const T*)a.v + t.s0 * a.ld_v + wk.hk * a.hs_v;
  const int keys = a.causal ? min(t.len, t.r0 + BM) : t.len;
  const int first = set * BN, step = SETS * BN;
  JaStage<T, DP, BN, BYTES, QW> sk, sv;
  sk.init(kb, a.ld_k, first, t.len, a.d);
  sv.init(vb, a.ld_v, first, t.len, a.dv);
  auto load = [&](int buf) {
    sk.load(ja_lds(lk + buf), step);
    sv.load(ja_lds(lv + buf), step);
  };
  if (first < keys) load(0);
  JaRows<T, DP, ja_keep<T, DP>> q, go;
  q.init((const T*)a.q + t.s0 * a.ld_q + head * a.hs_q, a.ld_q, q0, t.len, a.d);
  const int64_t out0 = (t.s0 * H + head) * a.dv;
  go.init((const T*)a.dout + out0, (int64_t)H * a.dv, q0, t.len, a.dv);
  const int64_t at = head * a.rows + t.s0 + (ok ? qi : 0);
  float delta = 0.f;
  if constexpr (GIVEN) {
    delta = a.delta[at];
  } else {
    JaRows<T, DP, false> out, low;
    out.init((const T*)a.out + out0, (int64_t)H * a.dv, q0, t.len, a.dv);
    low.init((const T*)(sizeof(T) == 2 ? a.out_low : a.out) + out0, (int64_t)H * a.dv, q0, t.len, a.dv);
#pragma unroll
    for (int s = 0; s < DP / F::K; ++s) {
      float x[16 / sizeof(T)], y[16 / sizeof(T)], z[16 / sizeof(T)];
      ja_floats<T>(out.at(s), x);
      ja_floats<T>(go.at(s), y);
      if (sizeof(T) == 2) ja_floats<T>(low.at(s), z);
#pragma unroll
      for (int i = 0; i < 16 / (int)sizeof(T); ++i) delta += (sizeof(T) == 2 ? x[i] + z[i] : x[i]) * y[i];
    }
    delta = half_sum(delta);
    if (ok && half == 0 && set == 0) a.delta[at] = delta;
  }
  const float lse = ok ? a.lse[at] : INFINITY;
  f32x16 acc[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i) acc[i] = f16_zero();
  ja_landed();
  for (int k0 = first, buf = 0; k0 - first < keys; k0 += step, buf = TILE - buf) {
    if (k0 + step < keys) load(TILE - buf);
    if (q0 < t.len && k0 < keys && !(a.causal && k0 > q0 + 31)) {
      const bool edge = k0 + BN > t.len || (a.causal && k0 + BN - 1 > q0);
      const int last = a.causal ? min(t.len - 1, qi) : t.len - 1;
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        f32x16 p = ja_scores(lk + buf, 32 * b, q);
        const f32x16 dp = ja_scores(lv + buf, 32 * b, go);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          p[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(p[r], a.scale_l2, -lse));
          if (edge && k0 + 32 * b + (r & 3) + 8 * (r >> 2) + 4 * half > last) p[r] = 0.f;
          p[r] *= dp[r] - delta;
        }
        const typename F::Rows ds(p);
#pragma unroll
        for (int i = 0; i < DT; ++i) acc[i] = ds.template mma<DP>(lk + buf, 32 * b, i, acc[i]);
      }
    }
    ja_landed();
  }
  if constexpr (SETS > 1) {
    constexpr int SUMS = QW * DT * 16 * 64;
    float* sums = reinterpret_cast<float*>(lds);
    if (set) ja_give<QW>(sums + (set - 1) * SUMS, acc);
    __syncthreads();
    if (set) return;
#pragma unroll
    for (int j = 0; j < SETS - 1; ++j) ja_take<QW>(sums + j * SUMS, acc);
  }
  T* row = dq + (int64_t)(ok ? qi - t.r0 : 0) * H * a.d;
#pragma unroll
  for (int i = 0; i < DT; ++i) ja_store_t<T>(row, 32 * i, a.d, acc[i], a.scale, ok);
}

// dK, dV: a workgroup per 32 QW key rows and key head, a wave per 32 keys and set, tiles of BQ query
// rows of each query head of the group in turn.  WANT: 1 = dV, 2 = dK, 3 = both in one launch;
// heads wider than 128 take a launch for each, as both results' accumulators and the
// keys' fragments do not fit the registers together.  bf16 at width 128 fits two waves a SIMD
// where the compiler is held to it (not with two sets and loads of 4 bytes, whose lanes have more
// addresses): 128 sequences of up to 996 rows, 4 heads, 334 us -> 192.
template <typename T, int DP, int BQ, int WANT, int BYTES, int QW, int SETS>
__device__ __forceinline__ void ja_dkv(const JaggedAttnArgs& a, unsigned block, u32x4_t* lds, float* lsum) {
  using F = JaFrag<T>;
  using Tile = JaTile<T, DP>;
  constexpr int BM = 32 * QW, NB = BQ / 32, DT = DP / 32, TILE = Tile::size(BQ);
  static_assert(SETS * 4 * TILE * 16 >= (SETS - 1) * QW * DT * 16 * 256, "the other sets' sums fit");
  const JaggedWork wk = jagged_work(a, 1, block);  // an item per key head
  if (wk.slot >= a.slots) return;
  const int hk = wk.hk, group = a.group, H = a.Hkv * group;
  const JaggedTile t = jagged_tile<BM, true>(a.offsets, a.B, a.rows, wk.slot);
  if (t.len == 0) return;
  T* dk = (T*)a.dk + ((t.s0 + t.r0) * a.Hkv + hk) * a.d;
  T* dv = (T*)a.dvv + ((t.s0 + t.r0) * a.Hkv + hk) * a.dv;
  if (t.none) {
    if (WANT & 2) ja_zero(dk, (int64_t)a.Hkv * a.d, min(BM, t.len - t.r0), a.d);
    if (WANT & 1) ja_zero(dv, (int64_t)a.Hkv * a.dv, min(BM, t.len - t.r0), a.dv);
    return;
  }
  const int lane = threadIdx.x & 63, wave = wave_id(), half = lane >> 5;
  const int set = SETS > 1 ? wave / QW : 0;
  u32x4_t *lq = lds + set * 4 * TILE, *lg = lq + 2 * TILE;
  float *ll = lsum + set * 4 * BQ, *ld = ll + 2 * BQ;
  const int k0 = t.r0 + 32 * (wave % QW), ki = k0 + (lane & 31);
  const bool ok = ki < t.len;
  const int first = a.causal ? t.r0 : 0, per = (t.len - first + BQ - 1) / BQ, n = per * group;
  int r0 = first, head = hk * group;  // the tile last loaded: query rows r0 on of a head
  JaStage<T, DP, BQ, BYTES, QW> sq, sg;
  auto next = [&]() {
    r0 += BQ;
    if (r0 >= t.len) {
      r0 = first;
      ++head;
      return true;
    }
    return false;
  };
  auto seek = [&]() {
    sq.seek((const T*)a.q + t.s0 * a.ld_q + head * a.hs_q, r0, t.len, a.d);
    sg.seek((const T*)a.dout + (t.s0 * H + head) * a.dv, r0, t.len, a.dv);
  };
  for (int i = 0; i < set; ++i) next();  // a set takes every SETS-th tile
  sq.init((const T*)a.q + t.s0 * a.ld_q + head * a.hs_q, a.ld_q, r0, t.len, a.d);
  sg.init((const T*)a.dout + (t.s0 * H + head) * a.dv, (int64_t)H * a.dv, r0, t.len, a.dv);
  auto load = [&](int buf) {
    sq.load(ja_lds(lq + buf * TILE), SETS * BQ);
    sg.load(ja_lds(lg + buf * TILE), SETS * BQ);
    // rows past the end come as zeros in all four (query rows are d apart at least, or the descriptor
    // would not end before them): their probabilities of 1 meet zeros
    const int64_t row = head * a.rows + t.s0 + r0;
    if (wave % QW == 0) ja_stage_floats<BQ>(a.lse + row, t.len - r0, ja_lds(ll + buf * BQ));
    if (wave % QW == 1) ja_stage_floats<BQ>(a.delta + row, t.len - r0, ja_lds(ld + buf * BQ));
  };
  if (set < n) load(0);
  JaRows<T, DP, ja_keep<T, DP>> k, v;
  k.init((const T*)a.k + t.s0 * a.ld_k + hk * a.hs_k, a.ld_k, k0, t.len, a.d);
  if (WANT & 2) v.init((const T*)a.v + t.s0 * a.ld_v + hk * a.hs_v, a.ld_v, k0, t.len, a.dv);
  f32x16 ak[WANT & 2 ? DT : 1], av[WANT & 1 ? DT : 1];
#pragma unroll
  for (int i = 0; i < DT; ++i) {
    if (WANT & 2) ak[i] = f16_zero();
    if (WANT & 1) av[i] = f16_zero();
  }
  ja_landed();
  for (int i = set, buf = 0; i - set < n; i += SETS, buf ^= 1) {
    const int now = r0;
    if (i + SETS < n) {
      bool moved = false;
#pragma unroll
      for (int j = 0; j < SETS; ++j) moved |= next();
      if (moved) seek();
      load(buf ^ 1);
    }
    if (k0 < t.len && i < n && !(a.causal && now + BQ - 1 < k0)) {
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const int rb = now + 32 * b;
        if (rb >= t.len || (a.causal && rb + 31 < k0)) continue;  // wave-uniform
        f32x16 p = ja_scores(lq + buf * TILE, 32 * b, k), ds;
        if (WANT & 2) ds = ja_scores(lg + buf * TILE, 32 * b, v);
        const bool edge = a.causal && rb < k0 + 31;
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          const int rr = 32 * b + 8 * r4 + 4 * half;
          const f4 l4 = *reinterpret_cast<const f4*>(ll + buf * BQ + rr), d4 = *reinterpret_cast<const f4*>(ld + buf * BQ + rr);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = 4 * r4 + e;
            p[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(p[r], a.scale_l2, -l4[e]));
            if (edge && now + rr + e < ki) p[r] = 0.f;
            if (WANT & 2) ds[r] = p[r] * (ds[r] - d4[e]);
          }
        }
        if (WANT & 1) {
          const typename F::Rows x(p);
#pragma unroll
          for (int j = 0; j < DT; ++j) av[j] = x.template mma<DP>(lg + buf * TILE, 32 * b, j, av[j]);
        }
        if (WANT & 2) {
          const typename F::Rows x(ds);
#pragma unroll
          for (int j = 0; j < DT; ++j) ak[j] = x.template mma<DP>(lq + buf * TILE, 32 * b, j, ak[j]);
        }
      }
    }
    ja_landed();
  }
  if constexpr (SETS > 1) {
    constexpr int SUMS = QW * DT * 16 * 64;
    float* sums = reinterpret_cast<float*>(lds);
    auto join = [&](auto& v) {
      if (set) ja_give<QW>(sums + (set - 1) * SUMS, v);
      __syncthreads();
      if (!set) {
#pragma unroll
        for (int j = 0; j < SETS - 1; ++j) ja_take<QW>(sums + j * SUMS, v);
      }
    };
    if (WANT & 1) join(av);
    if (WANT == 3) __syncthreads();
    if (WANT & 2) join(ak);
    if (set) return;
  }
  T* krow = dk + (int64_t)(ok ? ki - t.r0 : 0) * a.Hkv * a.d;
  T* vrow = dv + (int64_t)(ok ? ki - t.r0 : 0) * a.Hkv * a.dv;
#pragma unroll
  for (int j = 0; j < DT; ++j) {
    if (WANT & 2) ja_store_t<T>(krow, 32 * j, a.d, ak[j], a.scale, ok);
    if (WANT & 1) ja_store_t<T>(vrow, 32 * j, a.dv, av[j], 1.f, ok);
  }
}

template <typename T, int DP, int BN, int BYTES, int QW, int SETS>
__global__ __launch_bounds__(64 * QW * SETS) void jagged_attn_dq_kernel(JaggedAttnArgs a) {
  __shared__ u32x4_t lds[SETS * 4 * JaTile<T, DP>::size(BN)];
  ja_dq<T, DP, BN, BYTES, QW, SETS, false>(a, blockIdx.x, lds);
}
template <typename T, int DP, int BQ, int WANT, int BYTES, int QW, int SETS>
__global__ __launch_bounds__(64 * QW * SETS, sizeof(T) == 2 && DP == 128 && (BYTES == 16 || SETS == 1) ? 2 : 1)
    void jagged_attn_dkv_kernel(JaggedAttnArgs a) {
  __shared__ u32x4_t lds[SETS * 4 * JaTile<T, DP>::size(BQ)];
  __shared__ __attribute__((aligned(16))) float lsum[SETS * 4 * BQ];
  ja_dkv<T, DP, BQ, WANT, BYTES, QW, SETS>(a, blockIdx.x, lds, lsum);
}

// Few tiles: all passes in one launch, the key rows' workgroups first, after a launch for D.
// Alone, each leaves CUs idle behind its longest tiles; with many, a pass would only have the
// other's registers.  `keys` workgroups for each key pass.  In turn and joint (us, the backward's kernels
// together, causal ragged batches as at jagged_few):
//   fp32, width 64: 128 x 211 rows, 1 head (238 tiles) 51 and 46, 4 x 3,524, 4 heads (260) 580 and 385, 64 x 500, 4 heads
//   (776) 169 and 158; width 128: 81 and 65, 869 and 723, 347 and 332;
//   bf16, width 64: 4 x 3,524, 4 heads (260) 156 and 96, 32 x 2,028, 1 head (295) 105 and 73, 24 x 980, 4 heads (476) 72 and 73;
//   width 128: 8 x 2,400, 3 heads (243) 139 and 110, 32 x 2,028, 1 head (295) 124 and 112, 24 x 980, 4 heads (476) 86 and 108;
//   width 256: 479 and 356, 32 x 2,059, 1 head (299) 312 and 255, 24 x 980, 4 heads (476) 226 and 227.
template <typename T, int DP, int BN, int BYTES, int QW, int SETS>
__global__ __launch_bounds__(64 * QW * SETS) void jagged_attn_both_kernel(JaggedAttnArgs a, unsigned keys) {
  __shared__ u32x4_t lds[SETS * 4 * JaTile<T, DP>::size(BN)];
  __shared__ __attribute__((aligned(16))) float lsum[SETS * 4 * BN];
  if constexpr (DP <= 128) {
    if (blockIdx.x < keys)
      ja_dkv<T, DP, BN, 3, BYTES, QW, SETS>(a, blockIdx.x, lds, lsum);
    else
      ja_dq<T, DP, BN, BYTES, QW, SETS, true>(a, blockIdx.x - keys, lds);
  } else {
    if (blockIdx.x < keys)
      ja_dkv<T, DP, BN, 2, BYTES, QW, SETS>(a, blockIdx.x, lds, lsum);
    else if (blockIdx.x < 2 * keys)
      ja_dkv<T, DP, BN, 1, BYTES, QW, SETS>(a, blockIdx.x - keys, lds, lsum);
    else
      ja_dq<T, DP, BN, BYTES, QW, SETS, true>(a, blockIdx.x - 2 * keys, lds);
  }
}

// D: 16 lanes for each row and head.
template <typename T>
__global__ __launch_bounds__(256) void jagged_attn_delta_kernel(JaggedAttnArgs a) {
  const int64_t H = (int64_t)a.Hkv * a.group, i = (int64_t)blockIdx.x * 16 + threadIdx.x / 16;  // row * H + head
  if (i >= a.rows * H) return;
  constexpr int V = 16 / sizeof(T);
  float s = 0.f;
  for (int c = threadIdx.x % 16 * V; c < a.dv; c += 16 * V) {
    float x[V], y[V], z[V];
    ja_floats<T>(ja_fix16<T>(ja_load16<T>((const T*)a.out + i * a.dv, c, a.dv), c, a.dv), x);
    ja_floats<T>(ja_fix16<T>(ja_load16<T>((const T*)a.dout + i * a.dv, c, a.dv), c, a.dv), y);
    if (sizeof(T) == 2) ja_floats<T>(ja_fix16<T>(ja_load16<T>((const T*)a.out_low + i * a.dv, c, a.dv), c, a.dv), z);
#pragma unroll
    for (int j = 0; j < V; ++j) s += (sizeof(T) == 2 ? x[j] + z[j] : x[j]) * y[j];
  }
  s = sum16(s);
  if (threadIdx.x % 16 == 0) a.delta[i % H * a.rows + i / H] = s;
}

template <typename T, int DP, int BN, int BYTES, int QW, int SETS>
static void both_run(JaggedAttnArgs a, hipStream_t st) {
  a.slots = jagged_slots(a.rows, a.B, 32 * QW);
  const int64_t keys = jagged_grid(a.slots, a.Hkv, 1);
  hipLaunchKernelGGL((jagged_attn_delta_kernel<T>), dim3((unsigned)((a.rows * a.Hkv * a.group + 15) / 16)), dim3(256), 0, st, a);
  hipLaunchKernelGGL((jagged_attn_both_kernel<T, DP, BN, BYTES, QW, SETS>),
                     dim3((unsigned)(keys * (DP <= 128 ? 1 : 2) + jagged_grid(a.slots, a.Hkv, a.group))), dim3(64 * QW * SETS), 0, st, a, (unsigned)keys);
}
template <typename T, int DP, int BN, int BYTES, int QW, int SETS>
static void dq_run(JaggedAttnArgs a, hipStream_t st) {
  a.slots = jagged_slots(a.rows, a.B, 32 * QW);
  hipLaunchKernelGGL((jagged_attn_dq_kernel<T, DP, BN, BYTES, QW, SETS>), dim3((unsigned)jagged_grid(a.slots, a.Hkv, a.group)),
                     dim3(64 * QW * SETS), 0, st, a);
}
template <typename T, int DP, int BQ, int WANT, int BYTES, int QW, int SETS>
static void dkv_run(JaggedAttnArgs a, hipStream_t st) {
  a.slots = jagged_slots(a.rows, a.B, 32 * QW);
  hipLaunchKernelGGL((jagged_attn_dkv_kernel<T, DP, BQ, WANT, BYTES, QW, SETS>), dim3((unsigned)jagged_grid(a.slots, a.Hkv, 1)),
                     dim3(64 * QW * SETS), 0, st, a);
}
template <typename T, int DP, int BYTES>
static void bwd_shape(const JaggedAttnArgs& a, hipStream_t st) {
  const int H = a.Hkv * a.group;
  if constexpr (sizeof(T) == 4) {
    if constexpr (DP == 64) {
      if (jagged_few(a, H, 1))
        both_run<T, DP, 32, BYTES, 2, 4>(a, st);
      else if (jagged_few(a, H, 3))
        both_run<T, DP, 32, BYTES, 2, 2>(a, st);
      else {
        dq_run<T, DP, 32, BYTES, 2, 2>(a, st);
        if (jagged_few(a, a.Hkv, 1))
          dkv_run<T, DP, 32, 3, BYTES, 2, 4>(a, st);
        else
          dkv_run<T, DP, 32, 3, BYTES, 2, 2>(a, st);
      }
    } else if constexpr (DP == 128) {
      if (jagged_few(a, H, 3)) return both_run<T, DP, 32, BYTES, 2, 2>(a, st);
      dq_run<T, DP, 32, BYTES, 2, 2>(a, st);
      dkv_run<T, DP, 32, 3, BYTES, 2, 2>(a, st);
    } else {
      // (the joint kernel does not fit the scalar registers)
      dq_run<T, DP, 32, BYTES, 4, 1>(a, st);
      dkv_run<T, DP, 32, 1, BYTES, 4, 1>(a, st);
      dkv_run<T, DP, 32, 2, BYTES, 4, 1>(a, st);
    }
    return;
  } else {
    // (with loads of 4 bytes the joint kernel's addresses do not fit the scalar registers)
    if constexpr (BYTES == 16) {
      if (jagged_few(a, H, DP == 128 ? 1.f : 1.5f))
        return both_run<T, DP, 32, BYTES, 2, DP == 64 ? 4 : 2>(a, st);
    }
    if constexpr (DP == 64) {
      if (BYTES == 4 && jagged_few(a, H, 1.5f))
        dq_run<T, DP, 64, 4, 2, 4>(a, st);
      else
        dq_run<T, DP, 64, BYTES, 4, 1>(a, st);
      if (jagged_few(a, a.Hkv, 1.5f))
        dkv_run<T, DP, 32, 3, BYTES, 2, 4>(a, st);
      else
        dkv_run<T, DP, 64, 3, BYTES, 4, 1>(a, st);
    } else if constexpr (DP == 128) {
      if (jagged_few(a, H, 2.f))
        dq_run<T, DP, 32, BYTES, 4, 2>(a, st);
      else
        dq_run<T, DP, 32, BYTES, 4, 1>(a, st);
      if (jagged_few(a, a.Hkv, 2.75f))
        dkv_run<T, DP, 32, 3, BYTES, 2, 2>(a, st);
      else
        dkv_run<T, DP, 32, 3, BYTES, 4, 1>(a, st);
    } else {
      if (BYTES == 4 && jagged_few(a, H, 1.5f))
        dq_run<T, DP, 32, 4, 2, 2>(a, st);
      else
        dq_run<T, DP, 32, BYTES, 4, 1>(a, st);
      if (jagged_few(a, a.Hkv, 1.5f)) {
        dkv_run<T, DP, 32, 1, BYTES, 2, 2>(a, st);
        dkv_run<T, DP, 32, 2, BYTES, 2, 2>(a, st);
      } else {
        dkv_run<T, DP, 32, 1, BYTES, 4, 1>(a, st);
        dkv_run<T, DP, 32, 2, BYTES, 4, 1>(a, st);
      }
    }
  }
}
template <typename T, int BYTES>
static void bwd_width(const JaggedAttnArgs& a, hipStream_t st) {
  const int w = a.d > a.dv ? a.d : a.dv;
  if (w <= 64)
    bwd_shape<T, 64, BYTES>(a, st);
  else if (w <= 128)
    bwd_shape<T, 128, BYTES>(a, st);
  else
    bwd_shape<T, 256, BYTES>(a, st);
}
template <typename T>
static void bwd_any(const JaggedAttnArgs& a, hipStream_t st) {
  a.wide ? bwd_width<T, 16>(a, st) : bwd_width<T, 4>(a, st);
}

}  // namespace gr

extern "C" {

size_t gr_jagged_attn_bwd_workspace_size(int64_t rows, int H) {
  return rows > 0 && H > 0 ? (size_t)rows * (size_t)H * sizeof(float) : 0;
}

int gr_jagged_attn_bwd(const void* q, int64_t ld_q, int64_t hs_q, const void* k, int64_t ld_k, int64_t hs_k,
                       const void* v, int64_t ld_v, int64_t hs_v, const int64_t* offsets, int B, int64_t rows, int H,
                       int Hkv, int d, int dv, int causal, float scale, int bf16, const void* out,
                       const void* out_low, const float* lse,
                       const void* dout, void* dq, void* dk, void* dvv, void* workspace, size_t ws_bytes, void* stream) {
  gr::JaggedAttnArgs a{};
  a.q = q; a.ld_q = ld_q; a.hs_q = hs_q;
  a.k = k; a.ld_k = ld_k; a.hs_k = hs_k;
  a.v = v; a.ld_v = ld_v; a.hs_v = hs_v;
  a.offsets = offsets; a.B = B; a.rows = rows;
  a.Hkv = Hkv; a.d = d; a.dv = dv;
  a.causal = causal; a.scale = scale; a.scale_l2 = scale * 1.44269504f;
  a.out = const_cast<void*>(out); a.out_low = const_cast<void*>(out_low); a.lse = const_cast<float*>(lse);
  a.dout = dout; a.dq = dq; a.dk = dk; a.dvv = dvv; a.delta = (float*)workspace;
  if (gr::jagged_attn_check("gr_jagged_attn_bwd", a, H, bf16)) return 1;
  if (rows == 0) return 0;
  GR_REQUIRE(ld_q >= d, "gr_jagged_attn_bwd: query rows closer than their width");
  GR_REQUIRE(lse && dout && (out_low || !bf16) && dq && dk && dvv, "gr_jagged_attn_bwd: null pointer");
  GR_REQUIRE(workspace && ws_bytes >= gr_jagged_attn_bwd_workspace_size(rows, H), "gr_jagged_attn_bwd: workspace too small");
  const hipStream_t st = (hipStream_t)stream;
  GR_TIMED("jagged_attn_bwd", st, bf16 ? gr::bwd_any<__bf16>(a, st) : gr::bwd_any<float>(a, st));
  GR_LAUNCH_CHECK("gr_jagged_attn_bwd");
  return 0;
}

}  // extern "C"
