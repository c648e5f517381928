// Per-head softmax attention over jagged rows, forward (gr_jagged_attn_fwd).
//
//   S = scale Q K^T over the rows of one sequence (keys j <= i where causal),
//   O = softmax(S) V,  lse = log2 of the rows' sums for the backward pass
//
// One workgroup of four waves per 128 query rows and head, a wave per 32 rows.  One pass over
// the keys in tiles held in LDS (the next tile's loads in flight in registers meanwhile), with
// the running maximum and sum of each row: S^T = K Q^T puts a query row in a lane, so
// maximum, sum and rescaling are lane-local but for one exchange between lane halves.
#include <math.h>

#include "jagged_attn.h"

#include "../../include/gr_hstu.h"

namespace gr {

template <typename T, int DP, int BN>
__global__ __launch_bounds__(256) void jagged_attn_fwd_kernel(JaggedAttnArgs a) {
  using F = JaFrag<T>;
  constexpr int BM = 128, NB = BN / 32, DT = DP / 32;
  constexpr int SK = ja_row_stride<T>(DP), SV = ja_col_stride<T>(DP);
  __shared__ __attribute__((aligned(16))) T lk[BN * SK];
  __shared__ __attribute__((aligned(16))) T lv[BN * SV];
  const int64_t w = blockIdx.x;
  const int g = (int)(w % a.group);
  const int64_t ws = w / a.group;
  const int hk = (int)(ws / a.slots), head = hk * a.group + g;
  const int H = a.Hkv * a.group;
  // later tiles of a causal sequence have more keys: they go first
  const JaggedTile t = jagged_tile<BM>(a.offsets, a.B, a.rows, a.slots - 1 - ws % a.slots);
  if (t.len == 0) return;
  if (t.tail) {
    ja_zero((T*)a.out + ((t.s0 + t.r0) * H + head) * a.dv, (int64_t)H * a.dv, min(BM, t.len - t.r0), a.dv);
    return;
  }
  const int lane = threadIdx.x & 63, wave = wave_id(), half = lane >> 5;
  const int q0 = t.r0 + 32 * wave, qi = q0 + (lane & 31);
  const T* kb = (const T*)a.k + t.s0 * a.ld_k + hk * a.hs_k;
  const T* vb = (const T*)a.v + t.s0 * a.ld_v + hk * a.hs_v;
  const int keys = a.causal ? min(t.len, t.r0 + BM) : t.len;
  JaStage<T, DP, BN> sk, sv;
  sk.load(kb, a.ld_k, 0, t.len, a.d);
  sv.load(vb, a.ld_v, 0, t.len, a.dv);
  JaRows<T, DP, ja_keep<T, DP>> q;
  q.init((const T*)a.q + t.s0 * a.ld_q + head * a.hs_q, a.ld_q, q0, t.len, a.d);
  f32x16 o[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i) o[i] = f16_zero();
  float m = -INFINITY, l = 0.f;
  for (int k0 = 0; k0 < keys; k0 += BN) {
    __syncthreads();
    sk.store(lk, SK, k0, t.len, a.d);
    sv.store(lv, SV, k0, t.len, a.dv);
    __syncthreads();
    if (k0 + BN < keys) {
      sk.load(kb, a.ld_k, k0 + BN, t.len, a.d);
      sv.load(vb, a.ld_v, k0 + BN, t.len, a.dv);
    }
    // a wave whose rows are past the end, or before every key of the tile, has nothing here
    if (q0 >= t.len || (a.causal && k0 > q0 + 31)) continue;
    f32x16 s[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) s[b] = ja_scores(lk + 32 * b * SK, SK, q);
    if (k0 + BN > t.len || (a.causal && k0 + BN - 1 > q0)) {
      const int last = a.causal ? min(t.len - 1, qi) : t.len - 1;
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (k0 + 32 * b + (r & 3) + 8 * (r >> 2) + 4 * half > last) s[b][r] = -INFINITY;
    }
    float top = m;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, s[b][r]);
    top = fmaxf(top, swap_half(top));
    if (__any(top > m)) {  // rescale only where a maximum moved
      const float f = __builtin_amdgcn_exp2f((m - top) * a.scale_l2);
      l *= f;
#pragma unroll
      for (int i = 0; i < DT; ++i) o[i] *= f;
      m = top;
    }
    const float mc = m * a.scale_l2;
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
#pragma unroll
      for (int i = 0; i < DT; ++i) o[i] = p.mma(lv + 32 * b * SV, SV, 32 * i, o[i]);
    }
  }
  l += swap_half(l);
  const bool ok = qi < t.len;
  T* out = (T*)a.out + ((t.s0 + (ok ? qi : 0)) * H + head) * a.dv;
  const float inv = 1.f / l;
#pragma unroll
  for (int i = 0; i < DT; ++i) ja_store_t<T>(out, 32 * i, a.dv, o[i], inv, ok);
  if (a.lse && ok && half == 0) a.lse[head * a.rows + t.s0 + qi] = m * a.scale_l2 + __builtin_amdgcn_logf(l);
}

int jagged_attn_check(const char* what, const JaggedAttnArgs& a, int H) {
  GR_REQUIRE(a.B >= 0 && a.rows >= 0 && H >= 1 && a.Hkv >= 1 && H % a.Hkv == 0 && a.d >= 1 && a.d <= 256 &&
                 a.dv >= 1 && a.dv <= 256,
             "%s: bad sizes", what);
  GR_REQUIRE(a.scale > 0.f && a.scale < INFINITY, "%s: scale must be positive", what);
  GR_REQUIRE(a.rows == 0 || (a.q && a.k && a.v && a.offsets && a.out), "%s: null pointer", what);
  GR_REQUIRE(a.rows < (1ll << 31) && (a.rows / 32 + a.B + 1) * (int64_t)H < (1ll << 31), "%s: too many tiles", what);
  return 0;
}

template <typename T>
static void fwd_launch(const JaggedAttnArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)(a.slots * a.Hkv * a.group)), block(256);
  const int w = a.d > a.dv ? a.d : a.dv;
  constexpr int BN = sizeof(T) == 2 ? 64 : 32;
  if (w <= 64)
    hipLaunchKernelGGL((jagged_attn_fwd_kernel<T, 64, BN>), grid, block, 0, st, a);
  else if (w <= 128)
    hipLaunchKernelGGL((jagged_attn_fwd_kernel<T, 128, BN>), grid, block, 0, st, a);
  else
    hipLaunchKernelGGL((jagged_attn_fwd_kernel<T, 256, 32>), grid, block, 0, st, a);
}

}  // namespace gr

extern "C" int gr_jagged_attn_fwd(const void* q, int64_t ld_q, int64_t hs_q, const void* k, int64_t ld_k, int64_t hs_k,
                                  const void* v, int64_t ld_v, int64_t hs_v, const int64_t* offsets, int B, int64_t rows,
                                  int H, int Hkv, int d, int dv, int causal, float scale, int bf16, void* out, float* lse,
                                  void* stream) {
  gr::JaggedAttnArgs a{};
  a.q = q; a.ld_q = ld_q; a.hs_q = hs_q;
  a.k = k; a.ld_k = ld_k; a.hs_k = hs_k;
  a.v = v; a.ld_v = ld_v; a.hs_v = hs_v;
  a.offsets = offsets; a.B = B; a.rows = rows;
  a.Hkv = Hkv; a.d = d; a.dv = dv;
  a.causal = causal; a.scale = scale; a.scale_l2 = scale * 1.44269504f;
  a.out = out; a.lse = lse;
  if (gr::jagged_attn_check("gr_jagged_attn_fwd", a, H)) return 1;
  if (rows == 0) return 0;
  a.group = H / Hkv;
  a.slots = gr::jagged_slots(rows, B, 128);
  const hipStream_t st = (hipStream_t)stream;
  GR_TIMED("jagged_attn_fwd", st, bf16 ? gr::fwd_launch<__bf16>(a, st) : gr::fwd_launch<float>(a, st));
  GR_LAUNCH_CHECK("gr_jagged_attn_fwd");
  return 0;
}
