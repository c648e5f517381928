// Layer norm over the last dimension of row-strided rows, forward and backward.
//
//   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), xh = (x - mu) r, y = xh w + b
//   g = dy w:  dx = r (g - mean(g) - xh mean(g xh));  dw = sum_rows dy xh;  db = sum_rows dy
//
// Both passes are bound by memory: a row is read once, held in its team's registers (the
// variance from centred values, so no cancellation) and written once.  A team is 16 lanes,
// a wave or a workgroup, the smallest that holds the row in at most four 16-byte vectors
// per lane; longer rows run the looping kernels, which read a row again from cache for each
// reduction.  Vectors need no alignment beyond the element's.
// Sums are fp32.  The weight's and bias's gradients stay in each team's registers over its
// rows, meet in LDS in a fixed order, go to a partial row per workgroup and are summed by a
// second launch in a fixed order: no atomics, the same bits every run.
#include <type_traits>

#include "common.h"

#include "../../include/gr_hstu.h"

namespace gr {

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

// V elements of a row from column c (zero past D).
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
__device__ __forceinline__ float team_sum(float v, float (*buf)[4], int& slot) {
  v = sum16(v);
  if constexpr (TEAM == 16) return v;
  v += __shfl_xor(v, 16, 64);
  v += __shfl_xor(v, 32, 64);
  if constexpr (TEAM == 64) return v;
  float* b = buf[slot];
  slot ^= 1;
  if ((threadIdx.x & 63) == 0) b[threadIdx.x >> 6] = v;
  __syncthreads();
  return (b[0] + b[1]) + (b[2] + b[3]);
}

template <typename T, int TEAM, int NV>
__global__ __launch_bounds__(256) void ln_fwd_kernel(LnArgs a) {
  constexpr int V = 16 / sizeof(T), RPW = 256 / TEAM;
  __shared__ float buf[2][4];
  int slot = 0;
  const int lane = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
  const float inv = 1.f / (float)a.D;
  for (int64_t r0 = (int64_t)blockIdx.x * RPW; r0 < a.rows; r0 += (int64_t)gridDim.x * RPW) {
    const int64_t row = r0 + team;
    const bool in = row < a.rows;  // all of a team's threads agree
    const T* x = (const T*)a.x + (in ? row : r0) * a.ld_x;
    float v[NV][V];
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      ln_load<T, V>(x, (j * TEAM + lane) * V, a.D, v[j]);
#pragma unroll
      for (int i = 0; i < V; ++i) s += v[j][i];
    }
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
    if (!in) continue;
    T* y = (T*)a.y + row * a.ld_y;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * TEAM + lane) * V;
      float w[V], b[V];
      ln_param<V>(a.w, a.w16, c, a.D, 1.f, w);
      ln_param<V>(a.b, a.w16, c, a.D, 0.f, b);
#pragma unroll
      for (int i = 0; i < V; ++i) v[j][i] = v[j][i] * r * w[i] + b[i];
      ln_store<T, V>(y, c, a.D, v[j]);
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
  __shared__ float buf[2][4];
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
__global__ __launch_bounds__(256) void ln_bwd_kernel(LnArgs a) {
  constexpr int V = 16 / sizeof(T), RPW = 256 / TEAM;
  constexpr int SPAN = TEAM * NV * V;  // columns a team holds
  __shared__ float buf[2][4];
  __shared__ float meet[TEAM == 256 ? 1 : 4 * SPAN];
  int slot = 0;
  const int lane = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
  const float inv = 1.f / (float)a.D;
  float aw[NV][V], ab[NV][V];
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < V; ++i) aw[j][i] = ab[j][i] = 0.f;
  for (int64_t r0 = (int64_t)blockIdx.x * RPW; r0 < a.rows; r0 += (int64_t)gridDim.x * RPW) {
    const int64_t row = r0 + team;
    const bool in = row < a.rows;
    const int64_t at = in ? row : r0;
    const T *x = (const T*)a.x + at * a.ld_x, *dy = (const T*)a.dy + at * a.ld_dy;
    const float mu = a.stats[2 * at], r = a.stats[2 * at + 1];
    float xh[NV][V], g[NV][V];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      ln_load<T, V>(x, (j * TEAM + lane) * V, a.D, xh[j]);
      ln_load<T, V>(dy, (j * TEAM + lane) * V, a.D, g[j]);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * TEAM + lane) * V;
      float w[V];
      ln_param<V>(a.w, a.w16, c, a.D, 1.f, w);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        xh[j][i] = (xh[j][i] - mu) * r;
        if (in) {  // columns past D: dy loads as 0, so the sums take nothing from them
          aw[j][i] += g[j][i] * xh[j][i];
          ab[j][i] += g[j][i];
        }
        g[j][i] = c + i < a.D ? g[j][i] * w[i] : 0.f;
        s1 += g[j][i];
        s2 += g[j][i] * xh[j][i];
      }
    }
    if (!a.y) continue;  // the same for every thread
    s1 = team_sum<TEAM>(s1, buf, slot) * inv;
    s2 = team_sum<TEAM>(s2, buf, slot) * inv;
    if (!in) continue;
    T* dx = (T*)a.y + row * a.ld_y;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int i = 0; i < V; ++i) g[j][i] = r * (g[j][i] - s1 - xh[j][i] * s2);
      ln_store<T, V>(dx, (j * TEAM + lane) * V, a.D, g[j]);
    }
  }
  if (!a.part) return;
  // the workgroup's teams meet: within a wave by lane exchanges, across waves in LDS
  float* out = a.part + (int64_t)blockIdx.x * 2 * a.D;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if constexpr (TEAM < 256) __syncthreads();
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float s = k ? ab[j][i] : aw[j][i];
        const int c = (j * TEAM + lane) * V + i;
        if constexpr (TEAM == 256) {
          if (c < a.D) out[k * a.D + c] = s;
        } else {
          if constexpr (TEAM == 16) {
            s += __shfl_xor(s, 16, 64);
            s += __shfl_xor(s, 32, 64);
          }
          if ((threadIdx.x & 63) < TEAM) meet[(threadIdx.x >> 6) * SPAN + c] = s;
        }
      }
    if constexpr (TEAM < 256) {
      __syncthreads();
      for (int c = threadIdx.x; c < a.D; c += 256)
        out[k * a.D + c] = (meet[c] + meet[SPAN + c]) + (meet[2 * SPAN + c] + meet[3 * SPAN + c]);
    }
  }
}

template <typename T>
__global__ __launch_bounds__(256) void ln_bwd_loop_kernel(LnArgs a) {
  constexpr int V = 16 / sizeof(T);
  __shared__ float buf[2][4];
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
    s1 = team_sum<256>(s1, buf, slot) * inv;
    s2 = team_sum<256>(s2, buf, slot) * inv;
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

// dw (blockIdx.y == 0) and db (1): 32 columns per workgroup, 32 threads down the partial
// rows of each, then a fixed tree over them.
__global__ __launch_bounds__(1024) void ln_param_grad_kernel(const float* part, int n, int D, int w16, void* dw,
                                                             void* db) {
  __shared__ float s[32][33];
  const int c = blockIdx.x * 32 + (threadIdx.x & 31), g = threadIdx.x >> 5;
  float v = 0.f;
  if (c < D)
    for (int i = g; i < n; i += 32) v += part[((int64_t)i * 2 + blockIdx.y) * D + c];
  s[g][threadIdx.x & 31] = v;
  for (int h = 16; h >= 1; h >>= 1) {
    __syncthreads();
    if (g < h) s[g][threadIdx.x & 31] += s[g + h][threadIdx.x & 31];
  }
  void* out = blockIdx.y ? db : dw;
  if (g == 0 && c < D && out) {
    if (w16)
      ((__bf16*)out)[c] = (__bf16)s[0][threadIdx.x];
    else
      ((float*)out)[c] = s[0][threadIdx.x];
  }
}

// Workgroups of a backward pass: enough to fill the chip, few enough that the partial rows
// stay a small share of what is read.
static int64_t ln_bwd_groups(int64_t rows, int D, int team) {
  const int64_t want = (rows + 256 / team - 1) / (256 / team), most = team == 256 ? 512 : 1024;
  return want < most ? want : most;
}

// The team that holds a row of D elements and its vectors per thread (0: the loop).
static void ln_shape(int D, int bf16, int* team, int* nv) {
  const int V = bf16 ? 8 : 4;
  *team = D <= 64 * V ? 16 : D <= 256 * V ? 64 : 256;
  const int need = (D + *team * V - 1) / (*team * V);
  *nv = need <= 1 ? 1 : need <= 2 ? 2 : need <= 4 ? 4 : 0;
  if (*team == 64 && *nv == 1) *nv = 2;
  if (*team == 256 && *nv == 1) *nv = 2;
}

template <typename T>
static void ln_launch(const LnArgs& a, int team, int nv, int64_t groups, bool bwd, hipStream_t st) {
  const dim3 grid((unsigned)groups), block(256);
#define GR_LN_CASE(TEAM, NV)                                                              \
  if (team == TEAM && nv == NV) {                                                         \
    if (bwd)                                                                              \
      hipLaunchKernelGGL((ln_bwd_kernel<T, TEAM, NV>), grid, block, 0, st, a);            \
    else                                                                                  \
      hipLaunchKernelGGL((ln_fwd_kernel<T, TEAM, NV>), grid, block, 0, st, a);            \
    return;                                                                               \
  }
  GR_LN_CASE(16, 1)
  GR_LN_CASE(16, 2)
  GR_LN_CASE(16, 4)
  GR_LN_CASE(64, 2)
  GR_LN_CASE(64, 4)
  GR_LN_CASE(256, 2)
  GR_LN_CASE(256, 4)
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
  GR_REQUIRE(rows >= 0 && D >= 1 && types >= 0 && types < 4 && (rows == 0 || (x && y)), "gr_layer_norm_fwd: bad args");
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
  gr::ln_shape(D, types & 1, &team, &nv);
  const int64_t want = (rows + 256 / team - 1) / (256 / team), groups = want < 16384 ? want : 16384;
  GR_TIMED("layer_norm_fwd", st,
           (types & 1) ? gr::ln_launch<__bf16>(a, team, nv, groups, false, st)
                       : gr::ln_launch<float>(a, team, nv, groups, false, st));
  GR_LAUNCH_CHECK("gr_layer_norm_fwd");
  return 0;
}

size_t gr_layer_norm_bwd_workspace_size(int64_t rows, int D, int types) {
  if (rows < 0 || D < 1) return 0;
  int team, nv;
  gr::ln_shape(D, types & 1, &team, &nv);
  return (size_t)gr::ln_bwd_groups(rows, D, team) * 2 * (size_t)D * sizeof(float);
}

int gr_layer_norm_bwd(const void* dy, int64_t ld_dy, const void* x, int64_t ld_x, int64_t rows, int D,
                      const void* weight, int types, const float* stats, void* dx, int64_t ld_dx, void* dweight,
                      void* dbias, void* workspace, size_t ws_bytes, void* stream) {
  GR_REQUIRE(rows >= 0 && D >= 1 && types >= 0 && types < 4 && (rows == 0 || (dy && x && stats)),
             "gr_layer_norm_bwd: bad args");
  GR_REQUIRE(rows <= 1 || ((ld_x >= D || ld_x == 0) && (ld_dy >= D || ld_dy == 0) && (!dx || ld_dx >= D)),
             "gr_layer_norm_bwd: row strides below D");
  const bool params = dweight || dbias;
  GR_REQUIRE(!params || rows == 0 || (workspace && ws_bytes >= gr_layer_norm_bwd_workspace_size(rows, D, types)),
             "gr_layer_norm_bwd: workspace too small");
  if (!params && !dx) return 0;
  const hipStream_t st = (hipStream_t)stream;
  int team, nv;
  gr::ln_shape(D, types & 1, &team, &nv);
  const int64_t groups = gr::ln_bwd_groups(rows, D, team);
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
             hipLaunchKernelGGL(gr::ln_param_grad_kernel, dim3((unsigned)((D + 31) / 32), 2), dim3(1024), 0, st,
                                (const float*)workspace, (int)groups, D, types >> 1, dweight, dbias));
  GR_LAUNCH_CHECK("gr_layer_norm_bwd");
  return 0;
}

}  // extern "C"
