// AdamW over a tensor list with both moments held in 8 bits (gr_adamw8_step).
//
// A moment is an OCP e4m3 code times a power-of-two scale shared by 64 consecutive elements
// of one tensor.  Per element, with g the gradient and t the step's number:
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2          (fp32, no contraction)
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// and the parameter moves by the new moments before they are rounded.  The scale is the
// least power of two that keeps the block's largest magnitude within 448; each element
// is rounded down or up at random with the probability of its place between its two
// neighbours, so that the held moment's expectation is the moment.  Round-to-nearest would
// not do: v moves by 1 - b2 of itself a step (0.1 - 2 %) and half a step of e4m3 is
// 3 - 6 %, so it would stand still.  The random bits are a hash of the element's place and
// the step's number: replicas that see the same gradients round alike.  A nonzero v never
// becomes zero (m / eps would follow); below 2^-9 of the scale, 1/229,376 of the block's
// largest possible v, it is held at that value, which only shortens the steps of such elements.
// A block that holds an infinity or NaN gets a NaN scale: its moments are lost visibly.
//
// Bound by memory: 16.25 bytes an element (p and g read, p written, 1 byte a moment both ways and
// the scales).  35.9 M elements: 104 us, 5.6 TB/s, what a large copy reaches; 2.7 M: 12 us.  A lane
// holds 4 elements, so that codes move as dwords and a block is 16 lanes of one wave's row.
#include <cmath>

#include "common.h"

#include "../../include/gr_hstu.h"

namespace gr {
constexpr int ADAMW8_MAX = 64;    // tensors per launch (2.3 KB of kernel arguments)
constexpr int ADAMW8_SUB = 1024;  // elements per workgroup pass (4 per thread)
constexpr int ADAMW8_BLOCK = 64;  // elements per scale: one 16-lane row of 4 elements a lane

struct AdamW8Args {
  float* param[ADAMW8_MAX];
  const float* grad[ADAMW8_MAX];
  int64_t off[ADAMW8_MAX];  // first element in the moments, a multiple of ADAMW8_BLOCK
  int64_t n[ADAMW8_MAX];
  int first_chunk[ADAMW8_MAX + 1];
  int n_tensors;
  int advance;    // this launch writes step + 1
  int64_t chunk;  // elements per workgroup: a multiple of ADAMW8_SUB
  uint8_t* m;
  float* m_scale;
  uint8_t* v;
  float* v_scale;
  float* step;
  uint32_t* done;
  double lr, log2_b1, log2_b2;  // beta^t = 2^(t log2 beta): half a power's work
  float b1, c1, b2, c2, keep, eps;  // c = 1 - b, keep = 1 - lr wd, each rounded once from doubles
};

__device__ __forceinline__ uint32_t max16u(uint32_t x) {
  auto mx = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
  auto mov = [](uint32_t a, auto ctrl) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)a, decltype(ctrl)::value, 0xF, 0xF, true);
  };
  x = mx(x, mov(x, std::integral_constant<int, 0xB1>{}));   // quad_perm [1,0,3,2]
  x = mx(x, mov(x, std::integral_constant<int, 0x4E>{}));   // quad_perm [2,3,0,1]
  x = mx(x, mov(x, std::integral_constant<int, 0x141>{}));  // row_half_mirror
  x = mx(x, mov(x, std::integral_constant<int, 0x140>{}));  // row_mirror
  return x;
}

__device__ __forceinline__ uint32_t place_bits(uint32_t idx, uint32_t key) {
  uint32_t x = idx * 0x9E3779B9u + key;
  x = (x ^ (x >> 15)) * 0x3C6EF373u;
  x = (x ^ (x >> 13)) * 0xBB67AE85u;
  return x ^ (x >> 16);
}

// Four elements' decode: codes of one dword times the block's scale (exact: a power of two).
__device__ __forceinline__ void decode4(uint32_t c, float s, float (&x)[4]) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  const f2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
  x[0] = lo.x * s;
  x[1] = lo.y * s;
  x[2] = hi.x * s;
  x[3] = hi.y * s;
}

// Rounds the block's elements (4 per lane of a 16-lane row) with the 20 random bits of
// each; returns the lane's four codes and the block's scale.
template <bool POSITIVE>
__device__ __forceinline__ uint32_t encode4(const float (&x)[4], const uint32_t (&r)[4], float& scale) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t b = __float_as_uint(x[i]) & 0x7FFFFFFFu;
    top = b > top ? b : top;
  }
  top = max16u(top);
  // exponent of the largest magnitude rounded up to 1.75 x 2^n (448 = 1.75 x 2^8)
  uint32_t e = (top + 0x1FFFFFu) >> 23;
  e = e < 24u ? 24u : e;  // keeps scale and 1 / scale normal numbers
  const float inv = __uint_as_float((262u - e) << 23);
  float q[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float w = fabsf(x[i]) * inv;
    const float hi = __uint_as_float((__float_as_uint(w) + r[i]) & 0xFFF00000u);
    const float lo = floorf(w * 512.f + (float)r[i] * 0x1p-20f) * (1.f / 512.f);  // below the least normal
    q[i] = w < 0x1p-6f ? lo : hi;
    if (POSITIVE)
      q[i] = x[i] > 0.f && q[i] == 0.f ? 0x1p-9f : q[i];
    else
      q[i] = copysignf(q[i], x[i]);
  }
  const bool lost = top >= 0x7F800000u;
  scale = lost ? __uint_as_float(0x7FC00000u) : __uint_as_float((e - 8u) << 23);
  int c = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
  c = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], c, true);
  return lost ? 0u : (uint32_t)c;
}

__global__ __launch_bounds__(256) void adamw8_kernel(AdamW8Args a) {
#pragma clang fp contract(off)
  __shared__ float sc[3];
  const int w = blockIdx.x;
  int t = 0;  // the tensor of chunk w: the last whose first chunk is <= w (wave-uniform)
  for (int half = ADAMW8_MAX / 2; half >= 1; half /= 2)
    if (t + half < a.n_tensors && a.first_chunk[t + half] <= w) t += half;
  const int64_t n = a.n[t], off = a.off[t];
  const int64_t c0 = (int64_t)(w - a.first_chunk[t]) * a.chunk;
  const int64_t cend = n < c0 + a.chunk ? n : c0 + a.chunk;
  float* param = a.param[t];
  const float* grad = a.grad[t];
  const bool vec = ((reinterpret_cast<uintptr_t>(param) | reinterpret_cast<uintptr_t>(grad)) & 15) == 0;
  // whole 64-element blocks: the lanes of a tensor's last block past its end carry zeros
  const int64_t end = (cend + ADAMW8_BLOCK - 1) / ADAMW8_BLOCK * ADAMW8_BLOCK;
  float p[4], g[4], m[4], v[4], ms, vs;
  uint32_t mc, vc;
  auto load = [&](int64_t i) {
    if (i >= end) return;
    if (vec && i + 3 < n) {
      const float4 pv = *reinterpret_cast<const float4*>(param + i), gv = *reinterpret_cast<const float4*>(grad + i);
      p[0] = pv.x; p[1] = pv.y; p[2] = pv.z; p[3] = pv.w;
      g[0] = gv.x; g[1] = gv.y; g[2] = gv.z; g[3] = gv.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        p[e] = i + e < n ? param[i + e] : 0.f;
        g[e] = i + e < n ? grad[i + e] : 0.f;
      }
    }
    const int64_t at = off + i;
    mc = *reinterpret_cast<const uint32_t*>(a.m + at);
    vc = *reinterpret_cast<const uint32_t*>(a.v + at);
    ms = a.m_scale[at / ADAMW8_BLOCK];
    vs = a.v_scale[at / ADAMW8_BLOCK];
  };
  int64_t i = c0 + 4 * (int64_t)threadIdx.x;
  load(i);  // on its way while the step is read
  if (threadIdx.x == 0) {
    const float ts = a.step[0] + 1.f;
    sc[0] = ts;
    sc[1] = (float)(a.lr / (1.0 - exp2((double)ts * a.log2_b1)));
    sc[2] = (float)(1.0 / sqrt(1.0 - exp2((double)ts * a.log2_b2)));
  }
  __syncthreads();
  const float ts = sc[0], size = sc[1], root = sc[2];
  const uint32_t key = (uint32_t)ts * 0xA54FF53Bu;
  for (; i < end; i += ADAMW8_SUB) {
    decode4(mc, ms, m);
    decode4(vc, vs, v);
    const int64_t at = off + i;
    uint32_t rm[4], rv[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      m[e] = m[e] * a.b1 + g[e] * a.c1;
      v[e] = v[e] * a.b2 + g[e] * g[e] * a.c2;
      // square root and reciprocal to one step of fp32 each: the update's error stays some
      // 1e-7 of a step that is itself a small part of the parameter
      p[e] = p[e] * a.keep - size * (m[e] * __builtin_amdgcn_rcpf(__builtin_amdgcn_sqrtf(v[e]) * root + a.eps));
      const uint32_t h = place_bits((uint32_t)at + e, key);
      rm[e] = h & 0xFFFFFu;
      rv[e] = h >> 12;
    }
    if (vec && i + 3 < n) {
      *reinterpret_cast<float4*>(param + i) = float4{p[0], p[1], p[2], p[3]};
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + e < n) param[i + e] = p[e];
    }
    const uint32_t mn = encode4<false>(m, rm, ms), vn = encode4<true>(v, rv, vs);
    *reinterpret_cast<uint32_t*>(a.m + at) = mn;
    *reinterpret_cast<uint32_t*>(a.v + at) = vn;
    if ((threadIdx.x & 15) == 0) {
      a.m_scale[at / ADAMW8_BLOCK] = ms;
      a.v_scale[at / ADAMW8_BLOCK] = vs;
    }
    load(i + ADAMW8_SUB);
  }
  if (!a.advance) return;
  // The last workgroup to finish writes the step and re-arms the counters.  Workgroups count
  // in 64 groups and the last of each group once more: one counter for all is a queue of
  // some 10 ns a workgroup (2,660 of them: 36 us against 12).  Relaxed: an increment only
  // has to follow its workgroup's read of the step (consumed before the barrier above).
  if (threadIdx.x == 0) {
    const uint32_t n = gridDim.x, k = blockIdx.x % 64, mine = n / 64 + (k < n % 64), groups = n < 64 ? n : 64;
    uint32_t* sub = a.done + 16 * (1 + k);
    if (__hip_atomic_fetch_add(sub, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == mine - 1) {
      __hip_atomic_store(sub, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      if (__hip_atomic_fetch_add(a.done, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == groups - 1) {
        a.step[0] = ts;
        __hip_atomic_store(a.done, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
    }
  }
}
}  // namespace gr

extern "C" int gr_adamw8_step(float* const* params, const float* const* grads, const int64_t* offs,
                              const int64_t* numel, int n_tensors, uint8_t* exp_avg, float* exp_avg_scale,
                              uint8_t* exp_avg_sq, float* exp_avg_sq_scale, float* step, uint32_t* done,
                              double lr, double beta1, double beta2, double eps, double weight_decay,
                              void* stream) {
  GR_REQUIRE(n_tensors >= 0 && (n_tensors == 0 || (params && grads && offs && numel && exp_avg && exp_avg_scale &&
                                                   exp_avg_sq && exp_avg_sq_scale && step && done)),
             "gr_adamw8_step: bad args");
  GR_REQUIRE(((reinterpret_cast<uintptr_t>(exp_avg) | reinterpret_cast<uintptr_t>(exp_avg_sq)) & 3) == 0,
             "gr_adamw8_step: moments must be 4-byte aligned");
  const hipStream_t st = (hipStream_t)stream;
  int64_t total = 0;
  int last = -1;
  for (int i = 0; i < n_tensors; ++i) {
    GR_REQUIRE(numel[i] >= 0 && offs[i] >= 0 && offs[i] % gr::ADAMW8_BLOCK == 0 &&
                   (numel[i] == 0 || (params[i] && grads[i])),
               "gr_adamw8_step: tensor %d: bad pointer / size / offset", i);
    if (numel[i] > 0) last = i;
    total += numel[i];
  }
  if (last < 0) return 0;
  // >= ~4096 workgroups' worth of passes before a workgroup takes more than one
  int64_t subs = total / ((int64_t)gr::ADAMW8_SUB * 4096) + 1;
  subs = subs > 8 ? 8 : subs;
  const int64_t chunk = gr::ADAMW8_SUB * subs;
  gr::AdamW8Args a{};
  a.chunk = chunk;
  a.m = exp_avg;
  a.m_scale = exp_avg_scale;
  a.v = exp_avg_sq;
  a.v_scale = exp_avg_sq_scale;
  a.step = step;
  a.done = done;
  a.lr = lr;
  a.log2_b1 = std::log2(beta1);  // beta = 0: -inf, and 2^(t log2 beta) = 0
  a.log2_b2 = std::log2(beta2);
  a.b1 = (float)beta1;
  a.c1 = (float)(1.0 - beta1);
  a.b2 = (float)beta2;
  a.c2 = (float)(1.0 - beta2);
  a.keep = (float)(1.0 - lr * weight_decay);
  a.eps = (float)eps;
  int64_t chunks = 0;
  for (int i = 0; i <= last; ++i) {
    if (numel[i] == 0) continue;
    const int j = a.n_tensors++;
    a.param[j] = params[i];
    a.grad[j] = grads[i];
    a.off[j] = offs[i];
    a.n[j] = numel[i];
    a.first_chunk[j] = (int)chunks;
    chunks += (numel[i] + chunk - 1) / chunk;
    GR_REQUIRE(chunks < 0x7fffffff, "gr_adamw8_step: too many chunks");
    if (a.n_tensors < gr::ADAMW8_MAX && i < last) continue;
    a.first_chunk[a.n_tensors] = (int)chunks;
    a.advance = i == last;
    GR_TIMED("adamw8", st, hipLaunchKernelGGL(gr::adamw8_kernel, dim3((unsigned)chunks), dim3(256), 0, st, a));
    a.n_tensors = 0;
    chunks = 0;
  }
  GR_LAUNCH_CHECK("gr_adamw8_step");
  return 0;
}
