// Layer norm over the last dimension of row-strided rows, forward and backward.
//
//   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), xh = (x - mu) r, y = xh w + b
//   g = dy w:  dx = r (g - mean(g) - xh mean(g xh));  dw = sum_rows dy xh;  db = sum_rows dy
//
// Both passes are bound by memory: a row is read once, held in its team's registers (the
// variance from centred values, so no cancellation) and written once.  A team is the
// smallest power of two of threads, 16 to 1,024, that holds the row at 16 bytes a thread
// (twice that at 1,024), and loads its next row while it works on one; longer rows run the
// looping kernels, which read a row again from cache for each reduction.  Vectors need no
// alignment beyond the element's.  Sums are fp32.  The weight's and bias's gradients stay in
// each team's registers over its rows, meet in LDS in a fixed order, go to a partial row per
// workgroup and are summed by a second launch in a fixed order: no atomics, the same bits
// every run.  20,011 bf16 rows of 4,096: forward 62 us (5.3 TB/s), backward 110 + 7 (4.2 TB/s);
// 65,888 bf16 rows of 256: 14 and 21 + 4.  The looping backward, whose partial sums are in memory: 10,000 bf16
// rows of 16,384, 1,941 + 42 us (0.5 TB/s).
#include <type_traits>

#include "common.h"

#include "../../include/gr_hstu.h"

namespace gr {

constexpr int LN_COLUMNS = 1 << 29;  // rows are narrower: columns are counted in 32 bits, up to 2 D and a step

struct LnArgs {
  const void* x;
  int64_t ld_x;
  const void* dy;
  int64_t ld_dy;
  int64_t rows;
  int D;
  const void* w;
  const void* b;
  int w16;  // weight / bias are bf16
  float eps;
  float* stats;  // (rows, 2): mu, r
  void* y;       // forward: y; backward: dx (or NULL)
  int64_t ld_y;
  float* part;  // backward: (workgroups, 2, D) partial sums of dw and db, or NULL
};

template <typename T>
__device__ __forceinline__ float to_f(T v) { return (float)v; }

template <typename T, int V>
struct __attribute__((packed, aligned(sizeof(T)))) Pack {
  T v[V];
};

template <typename T>
struct Vec {  // 16 bytes of a row as they are in memory
  static constexpr int V = 16 / sizeof(T);
  T v[V];
  // from column c, zero past D
  __device__ __forceinline__ void load(const T* row, int c, int D) {
    if (c + V <= D) {
      const Pack<T, V> p = *reinterpret_cast<const Pack<T, V>*>(row + c);
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = p.v[i];
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = c + i < D ? row[c + i] : (T)0.f;
    }
  }
};
template <typename T, int V>
__device__ __forceinline__ void ln_load(const T* row, int c, int D, float (&o)[V]) {
  if (c + V <= D) {
    const Pack<T, V> p = *reinterpret_cast<const Pack<T, V>*>(row + c);
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = to_f(p.v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = c + i < D ? to_f(row[c + i]) : 0.f;
  }
}
template <typename T, int V>
__device__ __forceinline__ void ln_store(T* row, int c, int D, const float (&o)[V]) {
  if (c + V <= D) {
    Pack<T, V> p;
#pragma unroll
    for (int i = 0; i < V; ++i) p.v[i] = (T)o[i];
    *reinterpret_cast<Pack<T, V>*>(row + c) = p;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (c + i < D) row[c + i] = (T)o[i];
  }
}
template <int V>
__device__ __forceinline__ void ln_param(const void* w, int w16, int c, int D, float other, float (&o)[V]) {
  if (!w) {
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = other;
  } else if (w16) {
    ln_load<__bf16, V>((const __bf16*)w, c, D, o);
  } else {
    ln_load<float, V>((const float*)w, c, D, o);
  }
}

// Sum over a team of TEAM threads; every thread gets it.  `slot` alternates between two
// LDS areas, so one barrier per sum is enough.
template <int TEAM>
__device__ __forceinline__ float team_sum(float v, float (*buf)[16], int& slot) {
  v = sum16(v);
  if constexpr (TEAM >= 32) v += __shfl_xor(v, 16, 64);
  if constexpr (TEAM >= 64) v += __shfl_xor(v, 32, 64);
  if constexpr (TEAM > 64) {
    float* b = buf[slot];
    slot ^= 1;
    const int wave = threadIdx.x >> 6, first = wave / (TEAM / 64) * (TEAM / 64);
    if ((threadIdx.x & 63) == 0) b[wave] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < TEAM / 64; ++i) v += b[first + i];
  }
  return v;
}

// Two sums at once: one barrier.
template <int TEAM>
__device__ __forceinline__ void team_sum2(float& v, float& u, float (*buf)[32], int& slot) {
  v = sum16(v);
  u = sum16(u);
  if constexpr (TEAM >= 32) {
    v += __shfl_xor(v, 16, 64);
    u += __shfl_xor(u, 16, 64);
  }
  if constexpr (TEAM >= 64) {
    v += __shfl_xor(v, 32, 64);
    u += __shfl_xor(u, 32, 64);
  }
  if constexpr (TEAM > 64) {
    float* b = buf[slot];
    slot ^= 1;
    const int wave = threadIdx.x >> 6, first = wave / (TEAM / 64) * (TEAM / 64);
    if ((threadIdx.x & 63) == 0) {
      b[wave] = v;
      b[16 + wave] = u;
    }
    __syncthreads();
    v = u = 0.f;
#pragma unroll
    for (int i = 0; i < TEAM / 64; ++i) {
      v += b[first + i];
      u += b[16 + first + i];
    }
  }
}

constexpr int ln_threads(int team) { return team < 256 ? 256 : team; }

template <typename T, int TEAM, int NV>
__global__ __launch_bounds__(ln_threads(TEAM)) void ln_fwd_kernel(LnArgs a) {
  constexpr int V = 16 / sizeof(T), RPW = ln_threads(TEAM) / TEAM;
  __shared__ float buf[2][16];
  int slot = 0;
  const int lane = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
  const float inv = 1.f / (float)a.D;
  float w[NV][V], b[NV][V];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    ln_param<V>(a.w, a.w16, (j * TEAM + lane) * V, a.D, 1.f, w[j]);
    ln_param<V>(a.b, a.w16, (j * TEAM + lane) * V, a.D, 0.f, b[j]);
  }
  Vec<T> next[NV];
  auto load = [&](int64_t row) {
    const T* x = (const T*)a.x + (row < a.rows ? row : a.rows - 1) * a.ld_x;
#pragma unroll
    for (int j = 0; j < NV; ++j) next[j].load(x, (j * TEAM + lane) * V, a.D);
  };
  const int64_t step = (int64_t)gridDim.x * RPW;
  load((int64_t)blockIdx.x * RPW + team);
  for (int64_t r0 = (int64_t)blockIdx.x * RPW; r0 < a.rows; r0 += step) {
    const int64_t row = r0 + team;
    float v[NV][V];
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) s += v[j][i] = to_f(next[j].v[i]);
    if (r0 + step < a.rows) load(row + step);
    const float mu = team_sum<TEAM>(s, buf, slot) * inv;
    float q = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        v[j][i] = (j * TEAM + lane) * V + i < a.D ? v[j][i] - mu : 0.f;
        q += v[j][i] * v[j][i];
      }
    const float r = 1.f / sqrtf(team_sum<TEAM>(q, buf, slot) * inv + a.eps);
    if (row >= a.rows) continue;
    T* y = (T*)a.y + row * a.ld_y;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int i = 0; i < V; ++i) v[j][i] = v[j][i] * r * w[j][i] + b[j][i];
      ln_store<T, V>(y, (j * TEAM + lane) * V, a.D, v[j]);
    }
    if (a.stats && lane == 0) {
      a.stats[2 * row] = mu;
      a.stats[2 * row + 1] = r;
    }
  }
}

// Rows longer than the registers hold: one workgroup per row, read once for the mean, once
// for the variance and once for the output.
template <typename T>
__global__ __launch_bounds__(256) void ln_fwd_loop_kernel(LnArgs a) {
  constexpr int V = 16 / sizeof(T);
  __shared__ float buf[2][16];
  int slot = 0;
  const float inv = 1.f / (float)a.D;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = (const T*)a.x + row * a.ld_x;
    float s = 0.f, q = 0.f, v[V];
    for (int c = threadIdx.x * V; c < a.D; c += 256 * V) {
      ln_load<T, V>(x, c, a.D, v);
#pragma unroll
      for (int i = 0; i < V; ++i) s += v[i];
    }
    const float mu = team_sum<256>(s, buf, slot) * inv;
    for (int c = threadIdx.x * V; c < a.D; c += 256 * V) {
      ln_load<T, V>(x, c, a.D, v);
#pragma unroll
      for (int i = 0; i < V; ++i) q += c + i < a.D ? (v[i] - mu) * (v[i] - mu) : 0.f;
    }
    const float r = 1.f / sqrtf(team_sum<256>(q, buf, slot) * inv + a.eps);
    T* y = (T*)a.y + row * a.ld_y;
    for (int c = threadIdx.x * V; c < a.D; c += 256 * V) {
      float w[V], b[V];
      ln_load<T, V>(x, c, a.D, v);
      ln_param<V>(a.w, a.w16, c, a.D, 1.f, w);
      ln_param<V>(a.b, a.w16, c, a.D, 0.f, b);
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = (v[i] - mu) * r * w[i] + b[i];
      ln_store<T, V>(y, c, a.D, v);
    }
    if (a.stats && threadIdx.x == 0) {
      a.stats[2 * row] = mu;
      a.stats[2 * row + 1] = r;
    }
  }
}

template <typename T, int TEAM, int NV>
__global__ __launch_bounds__(ln_threads(TEAM)) void ln_bwd_kernel(LnArgs a) {
  constexpr int V = 16 / sizeof(T), THREADS = ln_threads(TEAM), RPW = THREADS / TEAM;
  constexpr int SPAN = TEAM * NV * V;  // columns a team holds
  __shared__ float buf[2][32];
  __shared__ float meet[RPW > 1 ? RPW * SPAN : 1];
  int slot = 0;
  const int lane = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
  const float inv = 1.f / (float)a.D;
  float w[NV][V], aw[NV][V], ab[NV][V];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    ln_param<V>(a.w, a.w16, (j * TEAM + lane) * V, a.D, 1.f, w[j]);
#pragma unroll
    for (int i = 0; i < V; ++i) aw[j][i] = ab[j][i] = 0.f;
  }
  // two rows are on their way while one is worked on: one alone left the memory waiting
  // (20,011 bf16 rows of 4,096: 131 against 109 us)
  struct Row {
    Vec<T> x[NV], g[NV];
    float mu, r;
  };
  auto load = [&](Row& n, int64_t row) {
    const int64_t at = row < a.rows ? row : a.rows - 1;
    const T *x = (const T*)a.x + at * a.ld_x, *dy = (const T*)a.dy + at * a.ld_dy;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      n.x[j].load(x, (j * TEAM + lane) * V, a.D);
      n.g[j].load(dy, (j * TEAM + lane) * V, a.D);
    }
    n.mu = a.stats[2 * at];
    n.r = a.stats[2 * at + 1];
  };
  const int64_t step = (int64_t)gridDim.x * RPW;
  auto work = [&](Row& n, int64_t row, bool more) {
    const bool in = RPW == 1 || row < a.rows;  // all of a team's threads agree
    const float mu = n.mu, r = n.r;
    float xh[NV][V], g[NV][V];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        xh[j][i] = (to_f(n.x[j].v[i]) - mu) * r;
        // columns past D: dy loads as 0, so no sum takes anything from them
        const float d = in ? to_f(n.g[j].v[i]) : 0.f;
        aw[j][i] += d * xh[j][i];
        ab[j][i] += d;
        g[j][i] = d * w[j][i];
        s1 += g[j][i];
        s2 += g[j][i] * xh[j][i];
      }
    if (more) load(n, row + 2 * step);
    if (!a.y) return;  // the same for every thread
    team_sum2<TEAM>(s1, s2, buf, slot);
    s1 *= inv;
    s2 *= inv;
    if (!in) return;
    T* dx = (T*)a.y + row * a.ld_y;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int i = 0; i < V; ++i) g[j][i] = r * (g[j][i] - s1 - xh[j][i] * s2);
      ln_store<T, V>(dx, (j * TEAM + lane) * V, a.D, g[j]);
    }
  };
  Row even, odd;
  const int64_t start = (int64_t)blockIdx.x * RPW;
  load(even, start + team);
  if (start + step < a.rows) load(odd, start + step + team);
  for (int64_t r0 = start; r0 < a.rows; r0 += 2 * step) {
    work(even, r0 + team, r0 + 2 * step < a.rows);
    if (r0 + step < a.rows) work(odd, r0 + step + team, r0 + 3 * step < a.rows);
  }
  if (!a.part) return;
  // the workgroup's teams meet in LDS, in their order
  float* out = a.part + (int64_t)blockIdx.x * 2 * a.D;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if constexpr (RPW > 1) __syncthreads();
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int c = (j * TEAM + lane) * V + i;
        if constexpr (RPW > 1)
          meet[team * SPAN + c] = k ? ab[j][i] : aw[j][i];
        else if (c < a.D)
          out[k * a.D + c] = k ? ab[j][i] : aw[j][i];
      }
    if constexpr (RPW > 1) {
      __syncthreads();
      for (int c = threadIdx.x; c < a.D; c += THREADS) {
        float s = meet[c];
        for (int t = 1; t < RPW; ++t) s += meet[t * SPAN + c];
        out[k * a.D + c] = s;
      }
    }
  }
}

template <typename T>
__global__ __launch_bounds__(256) void ln_bwd_loop_kernel(LnArgs a) {
  constexpr int V = 16 / sizeof(T);
  __shared__ float buf[2][32];
  int slot = 0;
  const float inv = 1.f / (float)a.D;
  float* out = a.part ? a.part + (int64_t)blockIdx.x * 2 * a.D : nullptr;
  if (out)
    for (int c = threadIdx.x; c < a.D; c += 256) out[c] = out[a.D + c] = 0.f;
  __syncthreads();
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *x = (const T*)a.x + row * a.ld_x, *dy = (const T*)a.dy + row * a.ld_dy;
    const float mu = a.stats[2 * row], r = a.stats[2 * row + 1];
    float s1 = 0.f, s2 = 0.f, v[V], g[V], w[V];
    for (int c = threadIdx.x * V; c < a.D; c += 256 * V) {
      ln_load<T, V>(x, c, a.D, v);
      ln_load<T, V>(dy, c, a.D, g);
      ln_param<V>(a.w, a.w16, c, a.D, 1.f, w);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float xh = (v[i] - mu) * r;
        if (out && c + i < a.D) {  // a column's partial sums belong to one thread
          out[c + i] += g[i] * xh;
          out[a.D + c + i] += g[i];
        }
        s1 += c + i < a.D ? g[i] * w[i] : 0.f;
        s2 += c + i < a.D ? g[i] * w[i] * xh : 0.f;
      }
    }
    if (!a.y) continue;
    team_sum2<256>(s1, s2, buf, slot);
    s1 *= inv;
    s2 *= inv;
    T* dx = (T*)a.y + row * a.ld_y;
    for (int c = threadIdx.x * V; c < a.D; c += 256 * V) {
      ln_load<T, V>(x, c, a.D, v);
      ln_load<T, V>(dy, c, a.D, g);
      ln_param<V>(a.w, a.w16, c, a.D, 1.f, w);
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = r * (g[i] * w[i] - s1 - (v[i] - mu) * r * s2);
      ln_store<T, V>(dx, c, a.D, v);
    }
  }
}

// The partial rows' sums: 16 of the 2 D columns (dw, then db) per workgroup, 64 threads down
// the partial rows of each, then a fixed tree over them.
__global__ __launch_bounds__(1024) void ln_param_grad_kernel(const float* part, int n, int D, int w16, void* dw,
                                                             void* db) {
  __shared__ float s[64][17];
  const int k = threadIdx.x & 15, g = threadIdx.x >> 4, c = blockIdx.x * 16 + k;
  float v = 0.f;
  if (c < 2 * D) {
#pragma unroll 8
    for (int i = g; i < n; i += 64) v += part[(int64_t)i * 2 * D + c];
  }
  s[g][k] = v;
  for (int h = 32; h >= 1; h >>= 1) {
    __syncthreads();
    if (g < h) s[g][k] += s[g + h][k];
  }
  void* out = c < D ? dw : db;
  const int at = c < D ? c : c - D;
  if (g == 0 && c < 2 * D && out) {
    if (w16)
      ((__bf16*)out)[at] = (__bf16)s[0][k];
    else
      ((float*)out)[at] = s[0][k];
  }
}

// The team that holds a row of D elements and its vectors per thread (0: the loop).
static void ln_shape(int D, int bf16, bool bwd, int* team, int* nv) {
  const int need = (D + (bf16 ? 8 : 4) - 1) / (bf16 ? 8 : 4);
  int t = 16;
  while (t < need && t < 1024) t *= 2;
  *team = t;
  // a bf16 backward row of two vectors a thread does not fit the registers of 1,024 threads
  *nv = need <= t ? 1 : need <= 2 * t && !(bf16 && bwd) ? 2 : 0;
}
// Rows a workgroup takes at a time, and the most workgroups: what the chip holds at once
// (forward), or half that, so that the partial rows stay a small share of what is read.
static int ln_rows_of(int team, int nv) { return nv == 0 ? 1 : gr::ln_threads(team) / team; }
static int64_t ln_groups(int64_t rows, int team, int nv, bool bwd) {
  const int rpw = ln_rows_of(team, nv), threads = nv == 0 ? 256 : ln_threads(team);
  const int64_t want = (rows + rpw - 1) / rpw, most = (int64_t)device_cus() * (bwd ? 1024 : 2048) / threads;
  return want < most ? want : most;
}

template <typename T>
static void ln_launch(const LnArgs& a, int team, int nv, int64_t groups, bool bwd, hipStream_t st) {
  const dim3 grid((unsigned)groups), block(nv ? ln_threads(team) : 256);
#define GR_LN_CASE(TEAM)                                                                            \
  if (team == TEAM && nv == 1) {                                                                    \
    if (bwd)                                                                                        \
      hipLaunchKernelGGL((ln_bwd_kernel<T, TEAM, 1>), grid, block, 0, st, a);                       \
    else                                                                                            \
      hipLaunchKernelGGL((ln_fwd_kernel<T, TEAM, 1>), grid, block, 0, st, a);                       \
    return;                                                                                         \
  }
  GR_LN_CASE(16)
  GR_LN_CASE(32)
  GR_LN_CASE(64)
  GR_LN_CASE(128)
  GR_LN_CASE(256)
  GR_LN_CASE(512)
  GR_LN_CASE(1024)
  if (nv == 2 && !bwd) {
    hipLaunchKernelGGL((ln_fwd_kernel<T, 1024, 2>), grid, block, 0, st, a);
    return;
  }
  if constexpr (sizeof(T) == 4) {
    if (nv == 2) {
      hipLaunchKernelGGL((ln_bwd_kernel<T, 1024, 2>), grid, block, 0, st, a);
      return;
    }
  }
#undef GR_LN_CASE
  if (bwd)
    hipLaunchKernelGGL(ln_bwd_loop_kernel<T>, grid, block, 0, st, a);
  else
    hipLaunchKernelGGL(ln_fwd_loop_kernel<T>, grid, block, 0, st, a);
}

}  // namespace gr

extern "C" {

int gr_layer_norm_fwd(const void* x, int64_t ld_x, int64_t rows, int D, const void* weight, const void* bias,
                      int types, float eps, void* y, int64_t ld_y, float* stats, void* stream) {
  GR_REQUIRE(rows >= 0 && D >= 1 && D < gr::LN_COLUMNS && types >= 0 && types < 4 && (rows == 0 || (x && y)),
             "gr_layer_norm_fwd: bad args");
  GR_REQUIRE(rows <= 1 || ((ld_x >= D || ld_x == 0) && ld_y >= D), "gr_layer_norm_fwd: row strides below D");
  if (rows == 0) return 0;
  const hipStream_t st = (hipStream_t)stream;
  gr::LnArgs a{};
  a.x = x;
  a.ld_x = ld_x;
  a.rows = rows;
  a.D = D;
  a.w = weight;
  a.b = bias;
  a.w16 = types >> 1;
  a.eps = eps;
  a.stats = stats;
  a.y = y;
  a.ld_y = ld_y;
  int team, nv;
  gr::ln_shape(D, types & 1, false, &team, &nv);
  const int64_t groups = gr::ln_groups(rows, team, nv, false);
  GR_TIMED("layer_norm_fwd", st,
           (types & 1) ? gr::ln_launch<__bf16>(a, team, nv, groups, false, st)
                       : gr::ln_launch<float>(a, team, nv, groups, false, st));
  GR_LAUNCH_CHECK("gr_layer_norm_fwd");
  return 0;
}

size_t gr_layer_norm_bwd_workspace_size(int64_t rows, int D, int types) {
  if (rows < 0 || D < 1) return 0;
  int team, nv;
  gr::ln_shape(D, types & 1, true, &team, &nv);
  return (size_t)gr::ln_groups(rows, team, nv, true) * 2 * (size_t)D * sizeof(float);
}

int gr_layer_norm_bwd(const void* dy, int64_t ld_dy, const void* x, int64_t ld_x, int64_t rows, int D,
                      const void* weight, int types, const float* stats, void* dx, int64_t ld_dx, void* dweight,
                      void* dbias, void* workspace, size_t ws_bytes, void* stream) {
  GR_REQUIRE(rows >= 0 && D >= 1 && D < gr::LN_COLUMNS && types >= 0 && types < 4 && (rows == 0 || (dy && x && stats)),
             "gr_layer_norm_bwd: bad args");
  GR_REQUIRE(rows <= 1 || ((ld_x >= D || ld_x == 0) && (ld_dy >= D || ld_dy == 0) && (!dx || ld_dx >= D)),
             "gr_layer_norm_bwd: row strides below D");
  const bool params = dweight || dbias;
  GR_REQUIRE(!params || rows == 0 || (workspace && ws_bytes >= gr_layer_norm_bwd_workspace_size(rows, D, types)),
             "gr_layer_norm_bwd: workspace too small");
  if (!params && !dx) return 0;
  const hipStream_t st = (hipStream_t)stream;
  int team, nv;
  gr::ln_shape(D, types & 1, true, &team, &nv);
  const int64_t groups = gr::ln_groups(rows, team, nv, true);
  if (rows > 0) {
    gr::LnArgs a{};
    a.x = x;
    a.ld_x = ld_x;
    a.dy = dy;
    a.ld_dy = ld_dy;
    a.rows = rows;
    a.D = D;
    a.w = weight;
    a.w16 = types >> 1;
    a.stats = const_cast<float*>(stats);
    a.y = dx;
    a.ld_y = ld_dx;
    a.part = params ? (float*)workspace : nullptr;
    GR_TIMED("layer_norm_bwd", st,
             (types & 1) ? gr::ln_launch<__bf16>(a, team, nv, groups, true, st)
                         : gr::ln_launch<float>(a, team, nv, groups, true, st));
  }
  if (params)
    GR_TIMED("layer_norm_bwd", st,
             hipLaunchKernelGGL(gr::ln_param_grad_kernel, dim3((unsigned)((2 * D + 15) / 16)), dim3(1024), 0, st,
                                (const float*)workspace, (int)groups, D, types >> 1, dweight, dbias));
  GR_LAUNCH_CHECK("gr_layer_norm_bwd");
  return 0;
}

}  // extern "C"
