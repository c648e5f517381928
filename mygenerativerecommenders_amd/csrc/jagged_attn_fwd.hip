// Per-head softmax attention over jagged rows, forward (gr_jagged_attn_fwd).
//
//   S = scale Q K^T over the rows of one sequence (keys j <= i where causal),
//   O = softmax(S) V,  lse = log2 of the rows' sums for the backward pass
//
// A workgroup per 32 QW query rows and head, a wave per 32 rows and set, SETS sets of waves that
// take the key tiles in turn and join their sums at the end.  One pass over the keys in tiles
// of BN held in LDS (the next tile on its way from memory meanwhile), with the running maximum
// and sum of each row: S^T = K Q^T puts a query row in a lane, so maximum, sum and rescaling
// are lane-local but for one exchange between lane halves.
//
// Bytes are no bound (q, k, v and out once: some 10 us where a launch takes 90); what is depends on
// the tiles.  Few of them: the longest sequence's chain of tiles (2 x 8,192 rows, 4 heads of 128,
// bf16: 141 us, 526 TFLOP/s).  Many: the vector work of the softmax, 16 exponentials a lane
// and tile beside 16 (width 64) to 64 matrix instructions, hidden only by other waves of the
// SIMD (128 x 996 rows, 4 heads of 128: 110 us, 415 TFLOP/s; with
// the rounding errors for a backward pass 168).  Tried and slower: the next tile's scores under this
// tile's softmax in one wave (54 us -> 71, 213 -> 246), as the registers cost it a wave; tiles staged
// through registers.
#include <math.h>

#include "jagged_attn.h"

#include "../../include/gr_hstu.h"

namespace gr {

// EXACT (bf16, for the backward pass): the probabilities' rounding errors go through the product
// with V too.  The backward pass subtracts sum(dO O) from dO V^T; left in O, they were a
// third of dQ's error beyond that of its own type.
template <typename T, int DP, int BN, int BYTES, int QW, int SETS, bool EXACT>
__global__ __launch_bounds__(64 * QW * SETS) void jagged_attn_fwd_kernel(JaggedAttnArgs a) {
  using F = JaFrag<T>;
  using Tile = JaTile<T, DP>;
  constexpr int BM = 32 * QW, NB = BN / 32, DT = DP / 32, TILE = Tile::size(BN);
  __shared__ u32x4_t lds[SETS * 4 * TILE];
  static_assert(sizeof(lds) >= (SETS - 1) * (QW * DT * 16 + 2 * QW) * 256, "the other sets' sums fit");
  const JaggedWork wk = jagged_work(a, a.group, blockIdx.x);
  if (wk.slot >= a.slots) return;
  const int head = wk.hk * a.group + wk.g, H = a.Hkv * a.group;
  const JaggedTile t = jagged_tile<BM, false>(a.offsets, a.B, a.rows, wk.slot);
  if (t.len == 0) return;
  if (t.none) {
    ja_zero((T*)a.out + ((t.s0 + t.r0) * H + head) * a.dv, (int64_t)H * a.dv, min(BM, t.len - t.r0), a.dv);
    return;
  }
  const int lane = threadIdx.x & 63, wave = wave_id(), half = lane >> 5;
  const int set = SETS > 1 ? wave / QW : 0;  // takes tiles set, set + SETS, ..
  u32x4_t *lk = lds + set * 4 * TILE, *lv = lk + 2 * TILE;
  const int q0 = t.r0 + 32 * (wave % QW), qi = q0 + (lane & 31);
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
  JaRows<T, DP, ja_keep<T, DP>> q;
  q.init((const T*)a.q + t.s0 * a.ld_q + head * a.hs_q, a.ld_q, q0, t.len, a.d);
  ja_landed();
  f32x16 o[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i) o[i] = f16_zero();
  float m = -INFINITY, l = 0.f;
  // Whether a row of the wave has a maximum so far from zero that m * scale_l2, rounded, is off by
  // more than a term can be (keys masked by a type's lowest value): the difference is taken first then.
  bool far = false;
  // every set makes the same number of rounds, the last one perhaps without a tile
  for (int k0 = first, buf = 0; k0 - first < keys; k0 += step, buf = TILE - buf) {
    if (k0 + step < keys) load(TILE - buf);
    // a wave whose rows are past the end, or before every key of the tile, has nothing here
    if (q0 < t.len && k0 < keys && !(a.causal && k0 > q0 + 31)) {
      f32x16 s[NB];
#pragma unroll
      for (int b = 0; b < NB; ++b) s[b] = ja_scores(lk + buf, 32 * b, q);
      if (k0 + BN > t.len || (a.causal && k0 + BN - 1 > q0)) {
        const int last = a.causal ? min(t.len - 1, qi) : t.len - 1;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (k0 + 32 * b + (r & 3) + 8 * (r >> 2) + 4 * half > last) s[b][r] = -INFINITY;
      }
      float top = -INFINITY;
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, s[b][r]);
      top = half_max(top);
      // Sums are relative to m, which follows the maximum only once that is 2^8 ahead: what is
      // summed stays below 2^8 times the rows, and the rescaling is rare.
      if (__builtin_expect(__any((top - m) * a.scale_l2 > 8.f), 0)) {
        top = fmaxf(top, m);
        // rows that have met nothing but -inf are asked too where another row of the wave runs ahead
        const float f = m == top ? 1.f : __builtin_amdgcn_exp2f((m - top) * a.scale_l2);
        m = top;
        l *= f;
#pragma unroll
        for (int i = 0; i < DT; ++i) o[i] *= f;
        far = __any(m > -INFINITY && fabsf(m) * a.scale_l2 > 0x1p20f);
      }
      float mc = m == -INFINITY ? 0.f : m * a.scale_l2;  // nothing but -inf so far: no terms
      if (__builtin_expect(far, 0)) {
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[b][r] -= m == -INFINITY ? 0.f : m;
        mc = 0.f;
      }
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[b][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][r], a.scale_l2, -mc));
          l += s[b][r];
        }
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const typename F::Rows p(s[b]);
        if constexpr (EXACT) {
          const typename F::Rows e = p.low(s[b]);
#pragma unroll
          for (int i = 0; i < DT; ++i) o[i] = p.template mma<DP, true>(lv + buf, 32 * b, i, o[i], &e);
        } else {
#pragma unroll
          for (int i = 0; i < DT; ++i) o[i] = p.template mma<DP>(lv + buf, 32 * b, i, o[i]);
        }
      }
    }
    ja_landed();
  }
  l = half_sum(l);
  if constexpr (SETS > 1) {
    constexpr int SUMS = QW * DT * 16 * 64;
    float *sums = reinterpret_cast<float*>(lds), *ml = sums + (SETS - 1) * SUMS + (wave % QW) * 128 + lane;
    if (set) {
      ja_give<QW>(sums + (set - 1) * SUMS, o);
      ml[(set - 1) * QW * 128] = m;
      ml[(set - 1) * QW * 128 + 64] = l;
    }
    __syncthreads();
    if (set) return;
#pragma unroll
    for (int j = 0; j < SETS - 1; ++j) {
      const float mj = ml[j * QW * 128], top = fmaxf(m, mj);
      const float f = m == top ? 1.f : __builtin_amdgcn_exp2f((m - top) * a.scale_l2);  // both may be -inf
      const float g = mj == top ? 1.f : __builtin_amdgcn_exp2f((mj - top) * a.scale_l2);
      ja_take<QW>(sums + j * SUMS, o, f, g);
      l = l * f + ml[j * QW * 128 + 64] * g;
      m = top;
    }
  }
  const bool ok = qi < t.len;
  const int64_t out0 = ((t.s0 + (ok ? qi : 0)) * H + head) * a.dv;
  T* low = sizeof(T) == 2 && a.out_low ? (T*)a.out_low + out0 : nullptr;
  const float inv = 1.f / l;
#pragma unroll
  for (int i = 0; i < DT; ++i) ja_store_t<T>((T*)a.out + out0, 32 * i, a.dv, o[i], inv, ok, low);
  // From 2^23 on a log-sum does not hold the sum any more, and the backward pass could not tell such a
  // row's probabilities: +inf makes them zero.
  if (a.lse && ok && half == 0)
    a.lse[head * a.rows + t.s0 + qi] =
        m > -INFINITY && fabsf(m * a.scale_l2) > 0x1p23f ? INFINITY : m * a.scale_l2 + __builtin_amdgcn_logf(l);
}

int jagged_attn_check(const char* what, JaggedAttnArgs& a, int H, int bf16) {
  const int least = bf16 ? 8 : 4;  // 16 bytes
  GR_REQUIRE(a.B >= 0 && a.rows >= 0 && H >= 1 && a.Hkv >= 1 && H % a.Hkv == 0 && a.d >= least && a.d <= 256 &&
                 a.dv >= least && a.dv <= 256,
             "%s: bad sizes", what);
  GR_REQUIRE(a.scale > 0.f && a.scale < INFINITY, "%s: scale must be positive", what);
  GR_REQUIRE(a.rows == 0 || (a.q && a.k && a.v && a.offsets && a.out), "%s: null pointer", what);
  GR_REQUIRE(a.rows < (1ll << 31) && (a.rows / 32 + a.B + 10) * (int64_t)H < (1ll << 31), "%s: too many tiles", what);
  const uintptr_t at = (uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.dout;
  const int64_t steps = a.ld_q | a.hs_q | a.ld_k | a.hs_k | a.ld_v | a.hs_v | a.d | a.dv;
  // LDS loads of 4 or 16 bytes: bf16 rows of even widths and strides on 4-byte boundaries
  const int64_t far = (int64_t)1 << 22;  // a tile's byte offsets stay below 2^31
  GR_REQUIRE(at % 4 == 0 && (!bf16 || steps % 2 == 0), "%s: bf16 rows must be pairs on 4-byte boundaries", what);
  GR_REQUIRE(a.rows == 0 || (a.ld_q >= 0 && a.ld_q < far && a.ld_k >= 0 && a.ld_k < far && a.ld_v >= 0 && a.ld_v < far),
             "%s: row strides outside [0, 2^22)", what);
  GR_REQUIRE((int64_t)H * a.dv < far, "%s: output rows of 2^22 elements and more", what);
  a.wide = at % 16 == 0 && steps % least == 0;
  a.group = H / a.Hkv;
    return 0;
}

template <typename T, int DP, int BN, int BYTES, int QW, int SETS>
static void fwd_run(JaggedAttnArgs a, hipStream_t st) {
  a.slots = jagged_slots(a.rows, a.B, 32 * QW);
  const dim3 grid((unsigned)jagged_grid(a.slots, a.Hkv, a.group)), block(64 * QW * SETS);
  if constexpr (sizeof(T) == 2) {
    if (a.out_low) {
      hipLaunchKernelGGL((jagged_attn_fwd_kernel<T, DP, BN, BYTES, QW, SETS, true>), grid, block, 0, st, a);
      return;
    }
  }
  hipLaunchKernelGGL((jagged_attn_fwd_kernel<T, DP, BN, BYTES, QW, SETS, false>), grid, block, 0, st, a);
}
template <typename T, int DP, int BYTES>
static void fwd_shape(const JaggedAttnArgs& a, hipStream_t st) {
  const int H = a.Hkv * a.group;
  if constexpr (sizeof(T) == 4) {
    if constexpr (DP == 64) {
      if (jagged_few(a, H, 1))
        fwd_run<T, DP, 32, BYTES, 2, 4>(a, st);
      else
        fwd_run<T, DP, 32, BYTES, 2, 2>(a, st);
    } else if constexpr (DP == 128) {
      fwd_run<T, DP, 32, BYTES, 2, 2>(a, st);
    } else {
      fwd_run<T, DP, 32, BYTES, 4, 1>(a, st);
    }
  } else if constexpr (DP <= 128) {
    if (jagged_few(a, H, DP == 64 ? 1.5f : 2.f))
      fwd_run<T, DP, 64, BYTES, DP == 64 ? 2 : 4, DP == 64 ? 4 : 2>(a, st);
    else
      fwd_run<T, DP, 64, BYTES, 4, 1>(a, st);
  } else if (jagged_few(a, H, 1.5f)) {
    fwd_run<T, DP, 32, BYTES, 2, 2>(a, st);
  } else {
    fwd_run<T, DP, 32, BYTES, 4, 1>(a, st);
  }
}
template <typename T, int BYTES>
static void fwd_width(const JaggedAttnArgs& a, hipStream_t st) {
  const int w = a.d > a.dv ? a.d : a.dv;
  if (w <= 64)
    fwd_shape<T, 64, BYTES>(a, st);
  else if (w <= 128)
    fwd_shape<T, 128, BYTES>(a, st);
  else
    fwd_shape<T, 256, BYTES>(a, st);
}
template <typename T>
static void fwd_any(const JaggedAttnArgs& a, hipStream_t st) {
  a.wide ? fwd_width<T, 16>(a, st) : fwd_width<T, 4>(a, st);
}

}  // namespace gr

extern "C" int gr_jagged_attn_fwd(const void* q, int64_t ld_q, int64_t hs_q, const void* k, int64_t ld_k, int64_t hs_k,
                                  const void* v, int64_t ld_v, int64_t hs_v, const int64_t* offsets, int B, int64_t rows,
                                  int H, int Hkv, int d, int dv, int causal, float scale, int bf16, void* out,
                                  void* out_low, float* lse, void* stream) {
  gr::JaggedAttnArgs a{};
  a.q = q; a.ld_q = ld_q; a.hs_q = hs_q;
  a.k = k; a.ld_k = ld_k; a.hs_k = hs_k;
  a.v = v; a.ld_v = ld_v; a.hs_v = hs_v;
  a.offsets = offsets; a.B = B; a.rows = rows;
  a.Hkv = Hkv; a.d = d; a.dv = dv;
  a.causal = causal; a.scale = scale; a.scale_l2 = scale * 1.44269504f;
  a.out = out; a.out_low = out_low; a.lse = lse;
  if (gr::jagged_attn_check("gr_jagged_attn_fwd", a, H, bf16)) return 1;
  if (rows == 0) return 0;
  const hipStream_t st = (hipStream_t)stream;
  GR_TIMED("jagged_attn_fwd", st, bf16 ? gr::fwd_any<__bf16>(a, st) : gr::fwd_any<float>(a, st));
  GR_LAUNCH_CHECK("gr_jagged_attn_fwd");
  return 0;
}
