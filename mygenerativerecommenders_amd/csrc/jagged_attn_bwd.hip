// Per-head softmax attention over jagged rows, backward (gr_jagged_attn_bwd).
//
// The probabilities are recomputed from the scores and the rows' log-sums, never stored:
//   P = 2^(S scale / ln 2 - lse),  dP = dO V^T,  D = sum(dO O),  dS = P (dP - D)
//   dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO
// Two launches, each with its result in registers and no atomics, so the bits do not depend
// on the order of workgroups: one over query rows (dQ, and D for the other), one over key
// rows (dK and dV, summed over the query heads that share them).  Seven products instead
// of the five that a single launch with atomic dQ sums would take.
#include <math.h>

#include "jagged_attn.h"

#include "../../include/gr_hstu.h"

namespace gr {

// dQ: one workgroup per 128 query rows and head, a wave per 32 rows, tiles of BN keys.
template <typename T, int DP, int BN>
__global__ __launch_bounds__(256) void jagged_attn_dq_kernel(JaggedAttnArgs a) {
  using F = JaFrag<T>;
  constexpr int BM = 128, NB = BN / 32, DT = DP / 32;
  constexpr int SK = ja_col_stride<T>(DP), SV = ja_row_stride<T>(DP);
  __shared__ __attribute__((aligned(16))) T lk[BN * SK];
  __shared__ __attribute__((aligned(16))) T lv[BN * SV];
  const int64_t w = blockIdx.x;
  const int g = (int)(w % a.group);
  const int64_t ws = w / a.group;
  const int hk = (int)(ws / a.slots), head = hk * a.group + g;
  const int H = a.Hkv * a.group;
  const JaggedTile t = jagged_tile<BM>(a.offsets, a.B, a.rows, a.slots - 1 - ws % a.slots);
  if (t.len == 0) return;
  T* dq = (T*)a.dq + ((t.s0 + t.r0) * H + head) * a.d;
  if (t.tail) {
    ja_zero(dq, (int64_t)H * a.d, min(BM, t.len - t.r0), a.d);
    return;
  }
  const int lane = threadIdx.x & 63, wave = wave_id(), half = lane >> 5;
  const int q0 = t.r0 + 32 * wave, qi = q0 + (lane & 31);
  const bool ok = qi < t.len;
  const T* kb = (const T*)a.k + t.s0 * a.ld_k + hk * a.hs_k;
  const T* vb = (const T*)a.v + t.s0 * a.ld_v + hk * a.hs_v;
  const int keys = a.causal ? min(t.len, t.r0 + BM) : t.len;
  JaStage<T, DP, BN> sk, sv;
  sk.load(kb, a.ld_k, 0, t.len, a.d);
  sv.load(vb, a.ld_v, 0, t.len, a.dv);
  JaRows<T, DP, ja_keep<T, DP>> q, go;
  q.init((const T*)a.q + t.s0 * a.ld_q + head * a.hs_q, a.ld_q, q0, t.len, a.d);
  const int64_t out0 = (t.s0 * H + head) * a.dv;
  go.init((const T*)a.dout + out0, (int64_t)H * a.dv, q0, t.len, a.dv);
  float delta = 0.f;
  {
    JaRows<T, DP, false> out;
    out.init((const T*)a.out + out0, (int64_t)H * a.dv, q0, t.len, a.dv);
#pragma unroll
    for (int s = 0; s < DP / F::K; ++s) {
      const u32x4_t x = out.at(s), y = go.at(s);
      T xs[16 / sizeof(T)], ys[16 / sizeof(T)];
      __builtin_memcpy(xs, &x, 16);
      __builtin_memcpy(ys, &y, 16);
#pragma unroll
      for (int i = 0; i < 16 / (int)sizeof(T); ++i) delta += (float)xs[i] * (float)ys[i];
    }
    delta += swap_half(delta);
  }
  const int64_t at = head * a.rows + t.s0 + (ok ? qi : 0);
  if (ok && half == 0) a.delta[at] = delta;
  const float lse = ok ? a.lse[at] : INFINITY;
  f32x16 acc[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i) acc[i] = f16_zero();
  for (int k0 = 0; k0 < keys; k0 += BN) {
    __syncthreads();
    sk.store(lk, SK, k0, t.len, a.d);
    sv.store(lv, SV, k0, t.len, a.dv);
    __syncthreads();
    if (k0 + BN < keys) {
      sk.load(kb, a.ld_k, k0 + BN, t.len, a.d);
      sv.load(vb, a.ld_v, k0 + BN, t.len, a.dv);
    }
    if (q0 >= t.len || (a.causal && k0 > q0 + 31)) continue;
    const bool edge = k0 + BN > t.len || (a.causal && k0 + BN - 1 > q0);
    const int last = a.causal ? min(t.len - 1, qi) : t.len - 1;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      f32x16 p = ja_scores(lk + 32 * b * SK, SK, q);
      const f32x16 dp = ja_scores(lv + 32 * b * SV, SV, go);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        p[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(p[r], a.scale_l2, -lse));
        if (edge && k0 + 32 * b + (r & 3) + 8 * (r >> 2) + 4 * half > last) p[r] = 0.f;
        p[r] *= dp[r] - delta;
      }
      const typename F::Rows ds(p);
#pragma unroll
      for (int i = 0; i < DT; ++i) acc[i] = ds.mma(lk + 32 * b * SK, SK, 32 * i, acc[i]);
    }
  }
  T* row = dq + (int64_t)(ok ? qi - t.r0 : 0) * H * a.d;
#pragma unroll
  for (int i = 0; i < DT; ++i) ja_store_t<T>(row, 32 * i, a.d, acc[i], a.scale, ok);
}

// dK, dV: one workgroup per 128 key rows and key head, a wave per 32 keys, tiles of BQ query
// rows of each query head of the group in turn.  WANT: 1 = dV, 2 = dK, 3 = both in one launch;
// heads wider than 128 take a launch for each, as both results' accumulators and the keys'
// fragments do not fit the registers together.
template <typename T, int DP, int BQ, int WANT>
__global__ __launch_bounds__(256) void jagged_attn_dkv_kernel(JaggedAttnArgs a) {
  using F = JaFrag<T>;
  constexpr int BM = 128, NB = BQ / 32, DT = DP / 32;
  constexpr int S = ja_col_stride<T>(DP);
  __shared__ __attribute__((aligned(16))) T lq[BQ * S];
  __shared__ __attribute__((aligned(16))) T lg[BQ * S];
  __shared__ __attribute__((aligned(16))) float ll[BQ], ld[BQ];
  const int64_t w = blockIdx.x;
  const int hk = (int)(w / a.slots), H = a.Hkv * a.group;
  const JaggedTile t = jagged_tile<BM>(a.offsets, a.B, a.rows, w % a.slots);
  if (t.len == 0) return;
  T* dk = (T*)a.dk + ((t.s0 + t.r0) * a.Hkv + hk) * a.d;
  T* dv = (T*)a.dvv + ((t.s0 + t.r0) * a.Hkv + hk) * a.dv;
  if (t.tail) {
    if (WANT & 2) ja_zero(dk, (int64_t)a.Hkv * a.d, min(BM, t.len - t.r0), a.d);
    if (WANT & 1) ja_zero(dv, (int64_t)a.Hkv * a.dv, min(BM, t.len - t.r0), a.dv);
    return;
  }
  const int lane = threadIdx.x & 63, wave = wave_id(), half = lane >> 5;
  const int k0 = t.r0 + 32 * wave, ki = k0 + (lane & 31);
  const bool ok = ki < t.len;
  JaRows<T, DP, ja_keep<T, DP>> k, v;
  k.init((const T*)a.k + t.s0 * a.ld_k + hk * a.hs_k, a.ld_k, k0, t.len, a.d);
  if (WANT & 2) v.init((const T*)a.v + t.s0 * a.ld_v + hk * a.hs_v, a.ld_v, k0, t.len, a.dv);
  f32x16 ak[WANT & 2 ? DT : 1], av[WANT & 1 ? DT : 1];
#pragma unroll
  for (int i = 0; i < DT; ++i) {
    if (WANT & 2) ak[i] = f16_zero();
    if (WANT & 1) av[i] = f16_zero();
  }
  const int first = a.causal ? t.r0 : 0, per = (t.len - first + BQ - 1) / BQ, n = per * a.group;
  JaStage<T, DP, BQ> sq, sg;
  float rl = 0.f, rd = 0.f;
  // tile i: query rows first + BQ (i % per) on of head hk * group + i / per
  auto load = [&](int i) {
    const int head = hk * a.group + i / per, r0 = first + BQ * (i % per);
    sq.load((const T*)a.q + t.s0 * a.ld_q + head * a.hs_q, a.ld_q, r0, t.len, a.d);
    sg.load((const T*)a.dout + (t.s0 * H + head) * a.dv, (int64_t)H * a.dv, r0, t.len, a.dv);
    if (threadIdx.x < BQ) {
      const int r = r0 + threadIdx.x;
      rl = r < t.len ? a.lse[head * a.rows + t.s0 + r] : INFINITY;  // no probability
      rd = r < t.len ? a.delta[head * a.rows + t.s0 + r] : 0.f;
    }
  };
  load(0);
  for (int i = 0; i < n; ++i) {
    const int r0 = first + BQ * (i % per);
    __syncthreads();
    sq.store(lq, S, r0, t.len, a.d);
    sg.store(lg, S, r0, t.len, a.dv);
    if (threadIdx.x < BQ) {
      ll[threadIdx.x] = rl;
      ld[threadIdx.x] = rd;
    }
    __syncthreads();
    if (i + 1 < n) load(i + 1);
    if (k0 >= t.len || (a.causal && r0 + BQ - 1 < k0)) continue;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const int rb = r0 + 32 * b;
      if (rb >= t.len || (a.causal && rb + 31 < k0)) continue;  // wave-uniform
      f32x16 p = ja_scores(lq + 32 * b * S, S, k), ds;
      if (WANT & 2) ds = ja_scores(lg + 32 * b * S, S, v);
      const bool edge = a.causal && rb < k0 + 31;
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        const int rr = 32 * b + 8 * r4 + 4 * half;
        const f4 l4 = *reinterpret_cast<const f4*>(ll + rr), d4 = *reinterpret_cast<const f4*>(ld + rr);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = 4 * r4 + e;
          p[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(p[r], a.scale_l2, -l4[e]));
          if (edge && r0 + rr + e < ki) p[r] = 0.f;
          if (WANT & 2) ds[r] = p[r] * (ds[r] - d4[e]);
        }
      }
      if (WANT & 1) {
        const typename F::Rows x(p);
#pragma unroll
        for (int j = 0; j < DT; ++j) av[j] = x.mma(lg + 32 * b * S, S, 32 * j, av[j]);
      }
      if (WANT & 2) {
        const typename F::Rows x(ds);
#pragma unroll
        for (int j = 0; j < DT; ++j) ak[j] = x.mma(lq + 32 * b * S, S, 32 * j, ak[j]);
      }
    }
  }
  T* krow = dk + (int64_t)(ok ? ki - t.r0 : 0) * a.Hkv * a.d;
  T* vrow = dv + (int64_t)(ok ? ki - t.r0 : 0) * a.Hkv * a.dv;
#pragma unroll
  for (int j = 0; j < DT; ++j) {
    if (WANT & 2) ja_store_t<T>(krow, 32 * j, a.d, ak[j], a.scale, ok);
    if (WANT & 1) ja_store_t<T>(vrow, 32 * j, a.dv, av[j], 1.f, ok);
  }
}

template <typename T>
static void bwd_launch(JaggedAttnArgs a, hipStream_t st) {
  const int w = a.d > a.dv ? a.d : a.dv;
  constexpr int BN = sizeof(T) == 2 ? 64 : 32;
  a.slots = jagged_slots(a.rows, a.B, 128);
  const dim3 gq((unsigned)(a.slots * a.Hkv * a.group)), gk((unsigned)(a.slots * a.Hkv)), block(256);
  if (w <= 64) {
    hipLaunchKernelGGL((jagged_attn_dq_kernel<T, 64, BN>), gq, block, 0, st, a);
    hipLaunchKernelGGL((jagged_attn_dkv_kernel<T, 64, BN, 3>), gk, block, 0, st, a);
  } else if (w <= 128) {
    hipLaunchKernelGGL((jagged_attn_dq_kernel<T, 128, 32>), gq, block, 0, st, a);
    hipLaunchKernelGGL((jagged_attn_dkv_kernel<T, 128, 32, 3>), gk, block, 0, st, a);
  } else {
    hipLaunchKernelGGL((jagged_attn_dq_kernel<T, 256, 32>), gq, block, 0, st, a);
    hipLaunchKernelGGL((jagged_attn_dkv_kernel<T, 256, 32, 1>), gk, block, 0, st, a);
    hipLaunchKernelGGL((jagged_attn_dkv_kernel<T, 256, 32, 2>), gk, block, 0, st, a);
  }
}

}  // namespace gr

extern "C" {

size_t gr_jagged_attn_bwd_workspace_size(int64_t rows, int H) {
  return rows > 0 && H > 0 ? (size_t)rows * (size_t)H * sizeof(float) : 0;
}

int gr_jagged_attn_bwd(const void* q, int64_t ld_q, int64_t hs_q, const void* k, int64_t ld_k, int64_t hs_k,
                       const void* v, int64_t ld_v, int64_t hs_v, const int64_t* offsets, int B, int64_t rows, int H,
                       int Hkv, int d, int dv, int causal, float scale, int bf16, const void* out, const float* lse,
                       const void* dout, void* dq, void* dk, void* dvv, void* workspace, size_t ws_bytes, void* stream) {
  gr::JaggedAttnArgs a{};
  a.q = q; a.ld_q = ld_q; a.hs_q = hs_q;
  a.k = k; a.ld_k = ld_k; a.hs_k = hs_k;
  a.v = v; a.ld_v = ld_v; a.hs_v = hs_v;
  a.offsets = offsets; a.B = B; a.rows = rows;
  a.Hkv = Hkv; a.d = d; a.dv = dv;
  a.causal = causal; a.scale = scale; a.scale_l2 = scale * 1.44269504f;
  a.out = const_cast<void*>(out); a.lse = const_cast<float*>(lse);
  a.dout = dout; a.dq = dq; a.dk = dk; a.dvv = dvv; a.delta = (float*)workspace;
  if (gr::jagged_attn_check("gr_jagged_attn_bwd", a, H)) return 1;
  if (rows == 0) return 0;
  GR_REQUIRE(lse && dout && dq && dk && dvv, "gr_jagged_attn_bwd: null pointer");
  GR_REQUIRE(workspace && ws_bytes >= gr_jagged_attn_bwd_workspace_size(rows, H), "gr_jagged_attn_bwd: workspace too small");
  a.group = H / Hkv;
  const hipStream_t st = (hipStream_t)stream;
  GR_TIMED("jagged_attn_bwd", st, bf16 ? gr::bwd_launch<__bf16>(a, st) : gr::bwd_launch<float>(a, st));
  GR_LAUNCH_CHECK("gr_jagged_attn_bwd");
  return 0;
}

}  // extern "C"
