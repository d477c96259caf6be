// Orthogonalisation of a batch of matrices by Newton-Schulz steps, and the optimizer step that uses it.
//
//   X0 = U / max(|U|_F, eps);  S = X X^T;  X <- (a I + b S + c S^2) X, a few times, on the side with fewer rows
//
// Each step applies p(x) = a x + b x^3 + c x^5 to the singular values, which (a, b, c) below push from (0, 1] to around 1.
// All products run on the tensor cores with fp16 operands and fp32 sums. fp16 and not bf16: every factor is bounded (|X| <=
// 1.21, |S| <= 1.46, |a I + b S + c S^2| <= a), so a constant scale of 512 keeps all of them inside fp16's range, and eight
// times finer rounding matters: a rounding of the first steps is amplified like the small singular values, by up to a^5 = 485.
// Error of the result (2-norm) against 64 bits on 768 x 2048 gradients with as much, a tenth and no white noise on a spectrum
// falling like 1 / i: 1.0e-3, 2.5e-3, 4.9e-3; with bf16 operands 9.3e-3, 2.0e-2, 3.9e-2. Empty directions raise roundings by as much:
// a 400 x 900 matrix of rank 1, 4, 60 ends 0.026, 0.011, 0.009 of its 2-norm off (bf16 0.31, 0.11, 0.10).
//
// An optimizer's master moves by learning rate times the result, so the results' error is 3e-6 of the master a step; to halve it,
// nearly every factor would need more bits (two fp16 parts, three times the products): left at fp16 by choice.
//
// A batch holds matrices whose shorter side is d and whose longer side is K; upright ones are transposed on the way in and
// out, so that the products see one layout: X [d, K] and symmetric factors [d, d], rows of whole 128 bytes.
//
// Four routes by size: one launch where everything fits one CTA's shared memory (ortho_small_kernel), all steps on the Gram
// matrix where rows are few and long (ortho_polynomial_kernel), else a launch per product, step by step or in pairs of steps
// (groups_of). The same call gives the same bits; other matrices in a batch may change the last ones of a matrix, by groups_of,
// gram_splits and the number of blocks that sum its squares. What bounds them: latency, then the start and end of launches (4.5 us
// each where products are short), and from about 1000 rows on the tensor cores under the power cap (a step of 16 matrices of 1536 x
// 1536 and 12 of 1536 x 4096: products 2.9 ms of 3.75, 0.92 PFLOP/s, 2.2 where each is timed by itself; one 5120 x 13696 0.98 to 1.06
// of the 1.41 that a GEMM holds).
#include "api.h"
#include "cluster.cuh"
#include "common.cuh"
#include "host.h"

#include <cuda_fp16.h>
#include <atomic>
#include <type_traits>

namespace aeris {

constexpr float NS_A = 3.4445f, NS_B = -4.7750f, NS_C = 2.0315f;
constexpr float NS_SCALE = 512.f;             // stored = NS_SCALE * value, for X and for the [d, d] factors

constexpr int NS_MAX_SIDE = 1 << 30;          // rows or columns of a matrix
constexpr int NS_PARTS = 1024;                // blocks per matrix that its squares are summed in, at most
constexpr int NS_GROUPS = ORTHO_GROUPS, NS_CLASSES = 2;

// ------------------------------------------------------------------------------------------------ in and out
// `count` matrices of one shape, from number `first` of their table on. Matrix i lies at element offsets[i] (checked against
// [0, numel) and for ascending order) or i * stride, with rows of pitch ld; its X [d, K] at x + i * x_stride with pitch ldx.
struct OrthoGroup {
  const long long* offsets;
  long long stride, x_stride;
  __half* x;
  double* partial;                            // [parts] per matrix
  int rows, cols, ld, ldx, behind, first, count, blocks, parts;      // behind: offsets[-1] is the matrix before the first one
  float rate;
};
struct OrthoGroups {
  OrthoGroup g[NS_GROUPS];
  long long numel;
  int n, aligned;                             // aligned: four elements from the buffers' starts on are one vector
  int* status;
};

struct OrthoPlace {
  int group, matrix, block;                   // matrix: its number in the table
  long long at;
  bool found, four;                           // four: rows are whole vectors of four
};
__device__ __forceinline__ long long ortho_size(const OrthoGroup& g) { return static_cast<long long>(g.rows) * g.cols; }
// Whether a matrix at `at` lies inside the buffers. Any 64-bit offset may be asked about: nothing is added to it.
__device__ __forceinline__ bool ortho_inside(const OrthoGroups& a, const OrthoGroup& g, long long at) {
  return at >= 0 && at <= a.numel - ortho_size(g);
}
__device__ __forceinline__ OrthoPlace ortho_place(const OrthoGroups& a) {
  OrthoPlace p;
  int b = blockIdx.x;
  p.group = 0;
  while (p.group + 1 < a.n && b >= a.g[p.group].count * a.g[p.group].blocks) b -= a.g[p.group].count * a.g[p.group].blocks, ++p.group;
  const OrthoGroup& g = a.g[p.group];
  p.matrix = g.first + b / g.blocks;
  p.block = b % g.blocks;
  p.found = true;
  if (!g.offsets) {
    p.at = p.matrix * g.stride;
  } else {
    p.at = g.offsets[p.matrix];
    p.found = ortho_inside(a, g, p.at) &&
              ((p.matrix == 0 && !g.behind) || g.offsets[p.matrix - 1] <= p.at - ortho_size(g));
    if (!p.found && threadIdx.x == 0) atomicCAS(a.status, 0, ERR_BOUNDS);
  }
  p.four = a.aligned && g.cols % 4 == 0 && g.ld % 4 == 0 && p.at % 4 == 0;
  return p;
}

// One warp: records a matrix of another group that shares elements with this one. One that lies outside is left out where its
// own block finds that.
__device__ __forceinline__ void ortho_apart(const OrthoGroups& a, const OrthoPlace& p) {
  if (!a.g[p.group].offsets || !p.found) return;
  const long long end = p.at + ortho_size(a.g[p.group]);
  for (int h = 0; h < a.n; ++h) {
    const OrthoGroup& g = a.g[h];
    if (h == p.group) continue;
    for (int i = threadIdx.x & 31; i < g.count; i += 32) {
      const long long at = g.offsets[g.first + i];
      if (ortho_inside(a, g, at) && at < end && at + ortho_size(g) > p.at) atomicCAS(a.status, 0, ERR_BOUNDS);
    }
  }
}

// What is orthogonalised: a tensor (fp32 or bf16), or the momentum of an optimizer.
struct OrthoInput {
  const void* x;
  int bf16;
  float *grad, *momentum;                     // optimizer: both set
  const double* norm_sq;
  float beta, grad_scale, max_norm;
  int nesterov, zero_grad;
};

__device__ __forceinline__ float step_scale(const OrthoInput& in) {      // as adamw_kernel
  float clip = 1.f;
  if (in.max_norm > 0.f && in.norm_sq) {
    const float c = in.max_norm / (static_cast<float>(sqrt(*in.norm_sq)) + 1.0e-6f);
    if (c < 1.f) clip = c;
  }
  return in.grad_scale * clip;
}
__device__ __forceinline__ float clean(float g) {
  return g != g ? 0.f : g > 3.0e38f ? 1.0e5f : g < -3.0e38f ? -1.0e5f : g;
}

__device__ __forceinline__ float in_value(const OrthoInput& in, long long e) {
  return in.bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(in.x)[e]) : reinterpret_cast<const float*>(in.x)[e];
}
__device__ __forceinline__ float4 in_value4(const OrthoInput& in, long long e) {
  if (!in.bf16) return *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(in.x) + e);
  const uint2 w = *reinterpret_cast<const uint2*>(reinterpret_cast<const __nv_bfloat16*>(in.x) + e);
  const float2 a = unpack_bf16x2(w.x), b = unpack_bf16x2(w.y);
  return make_float4(a.x, a.y, b.x, b.y);
}

// Sums of squares of one matrix, NS_PARTS at most, as good as in 64 bits (any fp32 values' squares add up without overflow). An
// optimizer's momentum is brought up to date on the way: M = beta M + (1 - beta) g; what is summed is M, or beta M + (1 -
// beta) g with nesterov. Bound by memory: 113 million elements of a step, 12 bytes each, 206 us (6.6 TB/s).
// The squares of a few vectors: in 32 bits where they neither overflow nor vanish there, which a sum between the bounds says (each
// term lost below has 2^-60 of it at most), for conversions to 64 bits and products in them are an eighth as fast.
template <int U> __device__ __forceinline__ double squares_of(const float4 (&u)[U]) {
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < U; ++k) s += u[k].x * u[k].x + u[k].y * u[k].y + (u[k].z * u[k].z + u[k].w * u[k].w);
  if (s > 1e-20f && s < 1e37f) return s;
  double d = 0;
#pragma unroll
  for (int k = 0; k < U; ++k) {
    d += static_cast<double>(u[k].x) * u[k].x + static_cast<double>(u[k].y) * u[k].y;
    d += static_cast<double>(u[k].z) * u[k].z + static_cast<double>(u[k].w) * u[k].w;
  }
  return d;
}

template <bool STEP>
__global__ void __launch_bounds__(256) ortho_squares_kernel(const OrthoGroups a, const OrthoInput in) {
  chain_point();
  const OrthoPlace p = ortho_place(a);
  const OrthoGroup& m = a.g[p.group];
  if (STEP && p.block == 0 && threadIdx.x < 32) ortho_apart(a, p);
  double sum = 0;
  if (p.found) {
    const float gs = STEP ? step_scale(in) : 0.f;
    auto value = [&](float g, float& mom) {
      g = clean(g * gs);
      mom = in.beta * mom + (1.f - in.beta) * g;
      return in.nesterov ? in.beta * mom + (1.f - in.beta) * g : mom;
    };
    const bool flat = m.ld == m.cols;
    const long long n = static_cast<long long>(m.rows) * m.cols;
    const long long step = m.blocks * 256ll, first = p.block * 256ll + threadIdx.x;
    if (p.four) {
      const int per_row = m.cols / 4;
      auto at = [&](long long v) { return flat ? p.at + 4 * v : p.at + v / per_row * m.ld + 4 * (v % per_row); };
      constexpr int U = STEP ? 2 : 4;         // vectors under way per thread
      for (long long v = first; v < n / 4; v += U * step) {
        float4 u[U], mo[U];
#pragma unroll
        for (int k = 0; k < U; ++k) {
          u[k] = mo[k] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (v + k * step >= n / 4) continue;
          const long long e = at(v + k * step);
          u[k] = STEP ? *reinterpret_cast<const float4*>(in.grad + e) : in_value4(in, e);
          if (STEP) mo[k] = *reinterpret_cast<const float4*>(in.momentum + e);
        }
#pragma unroll
        for (int k = 0; k < U; ++k) {
          if (STEP) {
            float4 &x = u[k], &y = mo[k];
            x = make_float4(value(x.x, y.x), value(x.y, y.y), value(x.z, y.z), value(x.w, y.w));
            if (v + k * step < n / 4) *reinterpret_cast<float4*>(in.momentum + at(v + k * step)) = y;
          }
        }
        sum += squares_of(u);
      }
    } else {
      auto at = [&](long long v) { return flat ? p.at + v : p.at + v / m.cols * m.ld + v % m.cols; };
      constexpr int U = 8;
      for (long long v = first; v < n; v += U * step) {
        float u[U], mo[U];
#pragma unroll
        for (int k = 0; k < U; ++k) {
          u[k] = mo[k] = 0.f;
          if (v + k * step >= n) continue;
          const long long e = at(v + k * step);
          u[k] = STEP ? in.grad[e] : in_value(in, e);
          if (STEP) mo[k] = in.momentum[e];
        }
        float4 q[U / 4];
#pragma unroll
        for (int k = 0; k < U; ++k) {
          if (STEP) {
            u[k] = value(u[k], mo[k]);
            if (v + k * step < n) in.momentum[at(v + k * step)] = mo[k];
          }
          reinterpret_cast<float*>(&q[k / 4])[k % 4] = u[k];
        }
        sum += squares_of(q);
      }
    }
  }
  __shared__ double red[8];
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 8; ++i) sum += red[i];
    m.partial[p.matrix * static_cast<long long>(m.parts) + p.block] = sum;
  }
}

// What an element u is multiplied by for X, as scale (pre u): one factor alone would be below fp32's normal range, and zero, where
// the norm is beyond 2^135, which elements within it reach. A norm that is no number stays one.
struct NormScale {
  float pre, scale;
  __device__ __forceinline__ NormScale(double norm, double eps) {
    pre = norm > 1e30 ? 0x1p-64f : 1.f;
    scale = static_cast<float>(NS_SCALE / ((norm > eps || norm != norm ? norm : eps) * pre));
  }
  __device__ __forceinline__ float operator()(float u) const { return scale * (pre * u); }
};

// Normed, scaled and rounded to fp16 into X [d, K], through shared memory where the matrix is upright: one 64 x 64 tile per
// block. An optimizer's value is computed again from gradient and momentum, which were read a moment before. Bound by memory
// like the pass before it: 113 million elements of a step, 14 bytes each, 188 us.
template <bool STEP>
__global__ void __launch_bounds__(256) ortho_pack_kernel(const OrthoGroups a, const OrthoInput in, double eps) {
  __shared__ float tile[64][65];
  __shared__ double red[8];
  chain_point();
  const OrthoPlace p = ortho_place(a);
  const OrthoGroup& m = a.g[p.group];
  if (!p.found) return;
  double sum = 0;
  for (int i = threadIdx.x; i < m.parts; i += 256) sum += m.partial[p.matrix * static_cast<long long>(m.parts) + i];
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = sum;
  __syncthreads();
  sum = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) sum += red[i];
  const double norm = sqrt(sum);
  const NormScale scale(norm, eps);
  const float gs = STEP ? step_scale(in) : 0.f;
  const int tiles_c = (m.cols + 63) / 64;
  const int r0 = p.block / tiles_c * 64, c0 = p.block % tiles_c * 64;
  const int tr = threadIdx.x >> 4, tc = (threadIdx.x & 15) * 4;
  __half* X = m.x + p.matrix * m.x_stride;
  const bool upright = m.rows > m.cols;
  auto value = [&](float g, float mom) {
    g = clean(g * gs);
    return scale(in.nesterov ? in.beta * mom + (1.f - in.beta) * g : mom);
  };
  if (p.four) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int r = r0 + tr + 16 * k, c = c0 + tc;
      float v[4] = {0.f, 0.f, 0.f, 0.f};
      if (r < m.rows && c < m.cols) {
        const long long e = p.at + static_cast<long long>(r) * m.ld + c;
        if (STEP) {
          const float4 g = *reinterpret_cast<const float4*>(in.grad + e);
          const float4 mo = *reinterpret_cast<const float4*>(in.momentum + e);
          v[0] = value(g.x, mo.x); v[1] = value(g.y, mo.y); v[2] = value(g.z, mo.z); v[3] = value(g.w, mo.w);
          if (in.zero_grad) *reinterpret_cast<float4*>(in.grad + e) = make_float4(0.f, 0.f, 0.f, 0.f);
        } else {
          const float4 u = in_value4(in, e);
          v[0] = scale(u.x); v[1] = scale(u.y); v[2] = scale(u.z); v[3] = scale(u.w);
        }
      }
      if (upright) {
#pragma unroll
        for (int j = 0; j < 4; ++j) tile[tr + 16 * k][tc + j] = v[j];
      } else if (r < m.rows && c < m.ldx) {
        __half2 h[2] = {__floats2half2_rn(v[0], v[1]), __floats2half2_rn(v[2], v[3])};
        *reinterpret_cast<uint2*>(X + static_cast<long long>(r) * m.ldx + c) = *reinterpret_cast<uint2*>(h);
      }
    }
  } else {                                    // element by element, a warp's side by side
    const int cc = threadIdx.x & 63, c = c0 + cc;
    const int first = threadIdx.x >> 6;
#pragma unroll 1
    for (int half = 0; half < 2; ++half) {
      float u[8], mo[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int r = r0 + first + 32 * half + 4 * k;
        u[k] = mo[k] = 0.f;
        if (r >= m.rows || c >= m.cols) continue;
        const long long e = p.at + static_cast<long long>(r) * m.ld + c;
        u[k] = STEP ? in.grad[e] : in_value(in, e);
        if (STEP) mo[k] = in.momentum[e];
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int rr = first + 32 * half + 4 * k, r = r0 + rr;
        const float v = STEP ? value(u[k], mo[k]) : scale(u[k]);
        if (STEP && in.zero_grad && r < m.rows && c < m.cols) in.grad[p.at + static_cast<long long>(r) * m.ld + c] = 0.f;
        if (upright) tile[rr][cc] = v;
        else if (r < m.rows && c < m.ldx) X[static_cast<long long>(r) * m.ldx + c] = __float2half_rn(v);
      }
    }
  }
  if (upright) {
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int r = c0 + tr + 16 * k, c = r0 + tc;          // row and column of X
      if (r < m.cols && c < m.ldx) {
        __half2 h[2] = {__floats2half2_rn(tile[tc][tr + 16 * k], tile[tc + 1][tr + 16 * k]),
                        __floats2half2_rn(tile[tc + 2][tr + 16 * k], tile[tc + 3][tr + 16 * k])};
        *reinterpret_cast<uint2*>(X + static_cast<long long>(r) * m.ldx + c) = *reinterpret_cast<uint2*>(h);
      }
    }
  }
}

// What becomes of the orthogonalised matrices: a bf16 tensor, or the update of an optimizer's weights.
struct OrthoOutput {
  __nv_bfloat16* out;
  float *master, *ema;                        // optimizer: master set
  __nv_bfloat16* weights;                     // may be null
  float decay, ema_beta;                      // master * decay - rate * X; ema_beta < 0: no running average
};

__device__ __forceinline__ void load_x4(const __half* p, float (&v)[4]) {
  const uint2 w = *reinterpret_cast<const uint2*>(p);
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
  v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
}

// X back in the matrices' own layout, upright ones through shared memory: one 64 x 64 tile per block. Bound by memory: 113
// million elements of a step, 22 bytes each, 390 us (6.4 TB/s).
template <bool STEP>
__global__ void __launch_bounds__(256) ortho_finish_kernel(const OrthoGroups a, const OrthoOutput o) {
  __shared__ float tile[64][65];
  chain_point();
  const OrthoPlace p = ortho_place(a);
  const OrthoGroup& m = a.g[p.group];
  if (!p.found || failed(a.status)) return;   // what a kernel that gave up left behind is not applied
  const int tiles_c = (m.cols + 63) / 64;
  const int r0 = p.block / tiles_c * 64, c0 = p.block % tiles_c * 64;
  const int tr = threadIdx.x >> 4, tc = (threadIdx.x & 15) * 4;
  const __half* X = m.x + p.matrix * m.x_stride;
  const bool upright = m.rows > m.cols;
  if (upright) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int r = c0 + tr + 16 * k, c = r0 + tc;
      if (r < m.cols && c < m.ldx) {
        float v[4];
        load_x4(X + static_cast<long long>(r) * m.ldx + c, v);
#pragma unroll
        for (int j = 0; j < 4; ++j) tile[tc + j][tr + 16 * k] = v[j];
      }
    }
    __syncthreads();
  }
  if (!p.four) {                              // element by element, a warp's side by side
    const int cc = threadIdx.x & 63, c = c0 + cc;
    if (c >= m.cols) return;
#pragma unroll 4
    for (int rr = threadIdx.x >> 6; rr < 64; rr += 4) {
      const int r = r0 + rr;
      if (r >= m.rows) break;
      const long long e = p.at + static_cast<long long>(r) * m.ld + c;
      const float v = (upright ? tile[rr][cc] : __half2float(X[static_cast<long long>(r) * m.ldx + c])) * (1.f / NS_SCALE);
      if (!STEP) {
        o.out[e] = __float2bfloat16_rn(v);
        continue;
      }
      const float w = o.master[e] * o.decay - m.rate * v;
      o.master[e] = w;
      if (o.weights) o.weights[e] = __float2bfloat16_rn(w);
      if (o.ema && o.ema_beta >= 0.f) o.ema[e] = w + o.ema_beta * (o.ema[e] - w);
    }
    return;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int r = r0 + tr + 16 * k, c = c0 + tc;
    if (r >= m.rows || c >= m.cols) continue;
    const long long e = p.at + static_cast<long long>(r) * m.ld + c;
    float v[4];
    if (upright) {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = tile[tr + 16 * k][tc + j];
    } else {
      load_x4(X + static_cast<long long>(r) * m.ldx + c, v);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] *= 1.f / NS_SCALE;
    if (!STEP) {
      *reinterpret_cast<uint2*>(o.out + e) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
      continue;
    }
    const float4 p4 = *reinterpret_cast<const float4*>(o.master + e);
    const float w[4] = {p4.x * o.decay - m.rate * v[0], p4.y * o.decay - m.rate * v[1], p4.z * o.decay - m.rate * v[2],
                        p4.w * o.decay - m.rate * v[3]};
    *reinterpret_cast<float4*>(o.master + e) = make_float4(w[0], w[1], w[2], w[3]);
    if (o.weights) *reinterpret_cast<uint2*>(o.weights + e) = make_uint2(pack_bf16x2(w[0], w[1]), pack_bf16x2(w[2], w[3]));
    if (o.ema && o.ema_beta >= 0.f) {
      float4 x = *reinterpret_cast<const float4*>(o.ema + e);
      x.x = w[0] + o.ema_beta * (x.x - w[0]); x.y = w[1] + o.ema_beta * (x.y - w[1]);
      x.z = w[2] + o.ema_beta * (x.z - w[2]); x.w = w[3] + o.ema_beta * (x.w - w[3]);
      *reinterpret_cast<float4*>(o.ema + e) = x;
    }
  }
}

// ------------------------------------------------------------------------------------------------ products
// C = alpha A B^T + beta R + gamma I for every matrix of a batch (B stored [K, N] with B_MN); fp16 in and out, fp32 sums.
// `sym`: the result is symmetric, only tiles on and below the diagonal are computed and the others are their mirror images.
// A batch has up to two classes of matrices, of longer sides of their own, so that all matrices with d rows share a launch.
//
// Two kernels of one scheme, a TMA producer, an issuer of tcgen05.mma, eight epilogue warps (two for the 32 rows of tensor memory
// each can read, with half of the columns) and two accumulators: 128 x 128 tiles on single CTAs, and 256 x 256 tiles on CTA
// pairs, each CTA staging its 128 rows of A and half of B's columns (csrc/gemm2.cu has the scheme), which need half the shared
// memory and L2 traffic per product. Results leave by 32 x 32 pieces through shared memory as tiled stores, their mirror images
// transposed by pairs of lanes on the way: with 2-byte stores of the mirror image the epilogue of a 256 x 256 tile took twice as
// long as its products (252 tiles of 1536: 55 us, 31 of which are products).
struct OrthoClass {
  int tiles, count, N, K;                     // tiles per matrix
  int a0, b0, c0;                             // first matrix of the class in the tensor maps of A, B and C
  // `splits` > 1 (128 x 128 tiles): so many CTAs share a tile's reduction and leave their sums in `partial`, one behind the other.
  // `low` > 0: A comes in two parts, and the reduction goes over B's rows with both, the second one `low` matrices on
  int splits, low;
};
struct OrthoGemm {
  OrthoClass cls[NS_CLASSES];
  int total, M, sym;                          // tiles in all
  float* partial;                             // splits: [matrix, tile, split, 128, 128]
  const __half* R;                            // null, or [matrices, M] rows of pitch ldr
  long long r_stride;
  int ldr;
  float alpha, beta, gamma;
  int* status;
};
struct OrthoMaps {
  CUtensorMap a[NS_CLASSES], b[NS_CLASSES], c[NS_CLASSES];
};

constexpr int OG_BK = 64, OG_STAGES = 5, OG_EPI_WARPS = 8, OG_THREADS = 64 + 32 * OG_EPI_WARPS;
constexpr int OG_OPERAND = 128 * OG_BK * 2;   // of one CTA, single or in a pair
constexpr int OG_STAGE = 2 * OG_OPERAND;
constexpr int OG_PIECE = 32 * 32 * 2;         // a 32 x 32 piece of C; two and their mirror images per epilogue warp
constexpr int OG_OUT = OG_STAGES * OG_STAGE + 256;
constexpr int OG_SMEM = (OG_OUT + 1023) / 1024 * 1024 + OG_EPI_WARPS * 4 * OG_PIECE + 1024;
static_assert(OG_SMEM <= 227 * 1024, "shared memory");

__device__ __forceinline__ void tma_load_3d(void* smem_dst, const CUtensorMap* m, uint64_t* bar, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
          smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* m, const void* smem_src, int c0, int c1, int c2) {   // no group yet
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(m)),
               "r"(smem_u32(smem_src)), "r"(c0), "r"(c1), "r"(c2)
               : "memory");
}
__host__ __device__ constexpr uint32_t make_idesc_fp16(int M, int N, int b_mn) {      // as make_idesc_bf16, formats 0 = fp16
  return (1u << 4) | (static_cast<uint32_t>(b_mn) << 16) | (static_cast<uint32_t>(N >> 3) << 17) |
         (static_cast<uint32_t>(M >> 4) << 24);
}

// Bounded waits that only their own time-out ends. Nothing here waits for another kernel's work, and a status word that is
// already set keeps results back (`keep`) without two CTAs or roles having to give up at the same place.
__device__ __forceinline__ bool own_wait(uint64_t* bar, uint32_t parity, int* status, int code) {
  if (mbar_wait(bar, parity, nullptr, 0)) return true;
  if (status) atomicCAS(status, 0, code);
  return false;
}
__device__ __forceinline__ bool own_poll(uint64_t* bar, uint32_t parity, int* status, int code) {
  if (mbar_wait_poll(bar, parity, nullptr, 0)) return true;
  if (status) atomicCAS(status, 0, code);
  return false;
}

// Tile `t` of the launch: class, matrix in it, and the tile's place, row by row or on and below the diagonal.
template <int TILE>
__device__ __forceinline__ void ortho_tile(const OrthoGemm& p, int t, int& cls, int& mat, int& ti, int& tj) {
  const int n0 = p.cls[0].tiles * p.cls[0].count;
  cls = t >= n0;
  t -= cls ? n0 : 0;
  const int per = cls ? p.cls[1].tiles : p.cls[0].tiles;
  mat = t / per;
  t -= mat * per;
  if (!p.sym) {
    const int n_tiles = ((cls ? p.cls[1].N : p.cls[0].N) + TILE - 1) / TILE;
    ti = t / n_tiles;
    tj = t - ti * n_tiles;
    return;
  }
  ti = static_cast<int>((sqrtf(8.f * t + 1.f) - 1.f) * 0.5f);
  while (ti * (ti + 1) / 2 > t) --ti;
  while ((ti + 1) * (ti + 2) / 2 <= t) ++ti;
  tj = t - ti * (ti + 1) / 2;
}

// A warp's 32 rows (from row0 on) of NCOL accumulator columns from `taddr` on, which are columns col0 .. of matrix `mat` of C.
// A piece's row of 64 bytes is swizzled by 16-byte chunks (64-byte swizzle of the tensor maps); in the mirror image lane l holds
// rows l & ~1 and l | 1 of column 2 j + (l & 1).
// `R`: this lane's row of R or null, `r` 64 values of it: two pieces are requested before the accumulator is waited for, the
// others while the one before them is worked on (d = 333: 7.3 us a launch with each requested when it is needed, 6.2).
struct Addend {
  const __half* R;
  uint4 r[2][4];
  int ld;
  __device__ void fetch(int col, int slot) {
    if (R && col < ld) {
#pragma unroll
      for (int j = 0; j < 4; ++j) r[slot][j] = *reinterpret_cast<const uint4*>(R + col + 8 * j);
    }
  }
  __device__ Addend(const OrthoGemm& p, int mat, int row, int col0) : R(nullptr), r{}, ld(p.ldr) {
    if (p.R && row < p.M) R = p.R + mat * p.r_stride + static_cast<long long>(row) * p.ldr;
    fetch(col0, 0);
    fetch(col0 + 32, 1);
  }
};
template <int NCOL>
__device__ __forceinline__ void ortho_epilogue(const OrthoGemm& p, const CUtensorMap* cmap, uint8_t* stage, uint32_t taddr, int mat,
                                               Addend& add, int row0, int col0, int N, bool keep, bool mirror, int lane,
                                               int& pieces) {
  const int row = row0 + lane;
  auto piece_of = [&](int c, uint4 (&r)[4]) {
    const int col = col0 + c;
    uint32_t v[32];
    tmem_ld32(taddr + c, v);
    tmem_wait_ld();
    float f[32];
#pragma unroll
    for (int j = 0; j < 32; ++j) f[j] = p.alpha * __uint_as_float(v[j]);
    if (add.R) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t w[4] = {r[j].x, r[j].y, r[j].z, r[j].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 r2 = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
          f[8 * j + 2 * i] += p.beta * r2.x;
          f[8 * j + 2 * i + 1] += p.beta * r2.y;
        }
      }
    }
    if (p.gamma != 0.f) {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (row == col + j) f[j] += p.gamma;
    }
    uint32_t h[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const __half2 x = __floats2half2_rn(f[2 * j], f[2 * j + 1]);
      h[j] = *reinterpret_cast<const uint32_t*>(&x);
    }
    uint8_t* piece = stage + (pieces & 1) * 2 * OG_PIECE;
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");      // the piece before the last has left
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *reinterpret_cast<uint4*>(piece + lane * 64 + ((i ^ ((lane >> 1) & 3)) << 4)) =
          make_uint4(h[4 * i], h[4 * i + 1], h[4 * i + 2], h[4 * i + 3]);
    if (mirror) {
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const uint32_t other = __shfl_xor_sync(0xffffffffu, h[j], 1);
        const uint32_t t = lane & 1 ? __byte_perm(other, h[j], 0x7632) : __byte_perm(h[j], other, 0x5410);
        const int rr = 2 * j + (lane & 1);
        *reinterpret_cast<uint32_t*>(piece + OG_PIECE + rr * 64 + (((lane >> 3) ^ (j & 3)) << 4) + (lane & 6) * 2) = t;
      }
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      if (keep && row0 < p.M) {
        tma_store_3d(cmap, piece, col, row0, mat);
        if (mirror) tma_store_3d(cmap, piece + OG_PIECE, row0, col, mat);
      }
      asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    }
    __syncwarp();
    ++pieces;
  };
#pragma unroll 1
  for (int c = 0; c < NCOL && col0 + c < N; c += 64) {
    piece_of(c, add.r[0]);
    if (c + 64 < NCOL) add.fetch(col0 + c + 64, 0);
    if (col0 + c + 32 >= N) break;
    piece_of(c + 32, add.r[1]);
    if (c + 64 < NCOL) add.fetch(col0 + c + 96, 1);
  }
}

// The tile that unit `unit` of a launch of single CTAs works on, and its blocks of the reduction. PARTS: `splits` or `low` are set.
template <bool PARTS> __device__ __forceinline__ int ortho_blocks(const OrthoGemm& p, int unit, int& kb0, int& kb1) {
  if (!PARTS) {
    kb0 = 0;
    kb1 = ((unit >= p.cls[0].tiles * p.cls[0].count ? p.cls[1].K : p.cls[0].K) + OG_BK - 1) / OG_BK;
    return unit;
  }
  const int splits = p.cls[0].splits;
  const int tile = splits > 1 ? unit / splits : unit;
  const int blocks = (p.cls[0].K + OG_BK - 1) / OG_BK * (p.cls[0].low ? 2 : 1);         // one class
  kb0 = 0;
  kb1 = blocks;
  if (splits > 1) {
    const int each = (blocks + splits - 1) / splits;
    kb0 = (unit - tile * splits) * each;
    kb1 = min(blocks, kb0 + each);
  }
  return tile;
}
// 32-bit sums of a lane's row
template <int NCOL> __device__ __forceinline__ void ortho_partial(float* to, uint32_t taddr) {
#pragma unroll 1
  for (int c = 0; c < NCOL; c += 32) {
    uint32_t v[32];
    tmem_ld32(taddr + c, v);
    tmem_wait_ld();
#pragma unroll
    for (int j = 0; j < 8; ++j)
      *reinterpret_cast<uint4*>(to + c + 4 * j) = make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
  }
}

template <int B_MN, bool PARTS>
__global__ void __launch_bounds__(OG_THREADS, 1) ortho_gemm_kernel(const __grid_constant__ OrthoMaps maps, const OrthoGemm p) {
  constexpr int TILE = 128;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + OG_STAGES * OG_STAGE);
  uint64_t* empty_bar = full_bar + OG_STAGES;
  uint64_t* tfull_bar = empty_bar + OG_STAGES;
  uint64_t* tempty_bar = tfull_bar + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty_bar + 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 32) {
    for (int c = 0; c < (p.cls[1].count ? 2 : 1); ++c) {
      prefetch_tmap(&maps.a[c]);
      prefetch_tmap(&maps.b[c]);
      prefetch_tmap(&maps.c[c]);
    }
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < OG_STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull_bar[a], 1);
      mbar_init(&tempty_bar[a], OG_EPI_WARPS);
    }
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 2 * TILE);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  chain_point();

  if (warp == 0) {
    if (elect_one_sync()) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int unit = blockIdx.x; unit < p.total && ok; unit += gridDim.x) {
        int cls, mat, ti, tj, kb0, kb1;
        ortho_tile<TILE>(p, ortho_blocks<PARTS>(p, unit, kb0, kb1), cls, mat, ti, tj);
        const CUtensorMap *ta = cls ? &maps.a[1] : &maps.a[0], *tb = cls ? &maps.b[1] : &maps.b[0];
        const int ma = mat + (cls ? p.cls[1].a0 : p.cls[0].a0), mb = mat + (cls ? p.cls[1].b0 : p.cls[0].b0);
        const int low_from = PARTS && p.cls[0].low ? (p.cls[0].K + OG_BK - 1) / OG_BK : kb1, low = PARTS ? p.cls[0].low : 0;
        for (int kb = kb0; kb < kb1; ++kb) {
          const int k = (kb < low_from ? kb : kb - low_from) * OG_BK, ma_now = ma + (kb < low_from ? 0 : low);
          if (!own_wait(&empty_bar[stage], phase ^ 1, p.status, ERR_TIMEOUT_EMPTY)) { ok = false; break; }
          uint8_t* sa = smem + stage * OG_STAGE;
          uint8_t* sb = sa + OG_OPERAND;
          mbar_expect_tx(&full_bar[stage], OG_STAGE);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            tma_load_3d(sa + j * 8192, ta, &full_bar[stage], k, ti * TILE + j * 64, ma_now);
            if (B_MN)
              tma_load_3d(sb + j * 8192, tb, &full_bar[stage], tj * TILE + j * 64, k, mb);
            else
              tma_load_3d(sb + j * 8192, tb, &full_bar[stage], k, tj * TILE + j * 64, mb);
          }
          if (++stage == OG_STAGES) { stage = 0; phase ^= 1; }
        }
      }
      // tiles that the issuer did not take (a stage never filled counts as there)
      for (int s = 0; s < OG_STAGES && !ok; ++s) {
        if (--stage < 0) { stage = OG_STAGES - 1; phase ^= 1; }
        if (!mbar_wait(&full_bar[stage], phase, nullptr, 0)) break;
      }
    }
  } else if (warp == 1) {
    if (elect_one_sync()) {
      constexpr uint32_t idesc = make_idesc_fp16(TILE, TILE, B_MN);
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int unit = blockIdx.x; unit < p.total && ok; unit += gridDim.x) {
        int kb0, kb1;
        ortho_blocks<PARTS>(p, unit, kb0, kb1);
        if (!own_wait(&tempty_bar[acc], acc_phase ^ 1, p.status, ERR_TIMEOUT_TMEM_EMPTY)) break;
        tc_fence_after();
        const uint32_t tmem_acc = tmem_base + acc * TILE;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!own_wait(&full_bar[stage], phase, p.status, ERR_TIMEOUT_FULL)) { ok = false; break; }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + stage * OG_STAGE), sb = sa + OG_OPERAND;
#pragma unroll
          for (int kk = 0; kk < OG_BK / 16; ++kk)
            umma_ss(tmem_acc, make_smem_desc(sa + kk * 32, 0, 1024),
                    B_MN ? make_smem_desc(sb + kk * 2048, 8192, 1024) : make_smem_desc(sb + kk * 32, 0, 1024), idesc,
                    kb > kb0 || kk > 0);
          tc_commit(&empty_bar[stage]);
          if (++stage == OG_STAGES) { stage = 0; phase ^= 1; }
        }
        if (!ok) break;
        tc_commit(&tfull_bar[acc]);
        if (++acc == 2) { acc = 0; acc_phase ^= 1; }
      }
      // the last products have completed before the tensor memory goes back (a stage never filled counts as done)
      if (--stage < 0) { stage = OG_STAGES - 1; phase ^= 1; }
      mbar_wait(&empty_bar[stage], phase, nullptr, 0);
    }
  } else {
    const int q = warp & 3, part = (warp - 2) >> 2;
    uint8_t* out = smem + (OG_OUT + 1023) / 1024 * 1024 + (warp - 2) * 4 * OG_PIECE;
    int acc = 0, pieces = 0;
    uint32_t acc_phase = 0;
    const bool keep = !failed(p.status);
    for (int unit = blockIdx.x; unit < p.total; unit += gridDim.x) {
      int cls, mat, ti, tj, kb0, kb1;
      ortho_tile<TILE>(p, ortho_blocks<PARTS>(p, unit, kb0, kb1), cls, mat, ti, tj);
      Addend add(p, mat, ti * TILE + q * 32 + lane, tj * TILE + part * (TILE / 2));
      if (!__all_sync(0xffffffffu, own_wait(&tfull_bar[acc], acc_phase, p.status, ERR_TIMEOUT_TMEM_FULL))) break;
      tc_fence_after();
      if (PARTS && p.partial)
        ortho_partial<TILE / 2>(p.partial + static_cast<long long>(unit) * (TILE * TILE) + (q * 32 + lane) * TILE + part * (TILE / 2),
                                tmem_base + acc * TILE + part * (TILE / 2) + (static_cast<uint32_t>(q * 32) << 16));
      else
        ortho_epilogue<TILE / 2>(p, cls ? &maps.c[1] : &maps.c[0], out,
                                 tmem_base + acc * TILE + part * (TILE / 2) + (static_cast<uint32_t>(q * 32) << 16),
                                 mat + (cls ? p.cls[1].c0 : p.cls[0].c0), add, ti * TILE + q * 32, tj * TILE + part * (TILE / 2),
                                 cls ? p.cls[1].N : p.cls[0].N, keep, p.sym && ti != tj, lane, pieces);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tempty_bar[acc]);
      if (++acc == 2) { acc = 0; acc_phase ^= 1; }
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem_base, 2 * TILE);
}

template <int B_MN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(OG_THREADS, 1)
ortho_gemm_pair_kernel(const __grid_constant__ OrthoMaps maps, const OrthoGemm p) {
  constexpr int TILE = 256;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + OG_STAGES * OG_STAGE);      // the leader's: both CTAs' bytes
  uint64_t* empty_bar = full_bar + OG_STAGES;
  uint64_t* tfull_bar = empty_bar + OG_STAGES;
  uint64_t* tempty_bar = tfull_bar + 2;                                               // the leader's: both CTAs' warps
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty_bar + 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t crank = cluster_ctarank();
  const int cluster = blockIdx.x >> 1, clusters = gridDim.x >> 1;
  if (threadIdx.x == 32) {
    for (int c = 0; c < (p.cls[1].count ? 2 : 1); ++c) {
      prefetch_tmap(&maps.a[c]);
      prefetch_tmap(&maps.b[c]);
      prefetch_tmap(&maps.c[c]);
    }
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < OG_STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull_bar[a], 1);
      mbar_init(&tempty_bar[a], 2 * OG_EPI_WARPS);
    }
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc2(tmem_slot, 2 * TILE);
    tmem_relinquish2();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  chain_point();

  if (warp == 0) {
    if (elect_one_sync()) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = cluster; tile < p.total && ok; tile += clusters) {
        int cls, mat, ti, tj;
        ortho_tile<TILE>(p, tile, cls, mat, ti, tj);
        const CUtensorMap *ta = cls ? &maps.a[1] : &maps.a[0], *tb = cls ? &maps.b[1] : &maps.b[0];
        const int ma = mat + (cls ? p.cls[1].a0 : p.cls[0].a0), mb = mat + (cls ? p.cls[1].b0 : p.cls[0].b0);
        const int kb_total = ((cls ? p.cls[1].K : p.cls[0].K) + OG_BK - 1) / OG_BK;
        const int m0 = ti * TILE + crank * 128, n0 = tj * TILE + crank * 128;
        for (int kb = 0; kb < kb_total; ++kb) {
          if (!own_poll(&empty_bar[stage], phase ^ 1, p.status, ERR_TIMEOUT_EMPTY)) { ok = false; break; }
          uint8_t* sa = smem + stage * OG_STAGE;
          uint8_t* sb = sa + OG_OPERAND;
          if (crank == 0) mbar_expect_tx(&full_bar[stage], 2 * OG_STAGE);
          const uint32_t fb = map_to_cta(smem_u32(&full_bar[stage]), 0);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            tma_load_3d_pair(sa + j * 8192, ta, fb, kb * OG_BK, m0 + j * 64, ma);
            if (B_MN)
              tma_load_3d_pair(sb + j * 8192, tb, fb, n0 + j * 64, kb * OG_BK, mb);
            else
              tma_load_3d_pair(sb + j * 8192, tb, fb, kb * OG_BK, n0 + j * 64, mb);
          }
          if (++stage == OG_STAGES) { stage = 0; phase ^= 1; }
        }
      }
      // tiles that the issuer did not take, of both CTAs (a stage never filled counts as there)
      for (int s = 0; s < OG_STAGES && !ok && crank == 0; ++s) {
        if (--stage < 0) { stage = OG_STAGES - 1; phase ^= 1; }
        if (!mbar_wait_poll(&full_bar[stage], phase, nullptr, 0)) break;
      }
    }
  } else if (warp == 1) {
    if (crank == 0 && elect_one_sync()) {
      constexpr uint32_t idesc = make_idesc_fp16(TILE, TILE, B_MN);
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int tile = cluster; tile < p.total && ok; tile += clusters) {
        const int kb_total = ((tile >= p.cls[0].tiles * p.cls[0].count ? p.cls[1].K : p.cls[0].K) + OG_BK - 1) / OG_BK;
        if (!own_poll(&tempty_bar[acc], acc_phase ^ 1, p.status, ERR_TIMEOUT_TMEM_EMPTY)) break;
        tc_fence_after();
        const uint32_t tmem_acc = tmem_base + acc * TILE;
        for (int kb = 0; kb < kb_total; ++kb) {
          if (!own_poll(&full_bar[stage], phase, p.status, ERR_TIMEOUT_FULL)) { ok = false; break; }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + stage * OG_STAGE), sb = sa + OG_OPERAND;
#pragma unroll
          for (int kk = 0; kk < OG_BK / 16; ++kk)
            umma2_ss(tmem_acc, make_smem_desc(sa + kk * 32, 0, 1024),
                     B_MN ? make_smem_desc(sb + kk * 2048, 8192, 1024) : make_smem_desc(sb + kk * 32, 0, 1024), idesc,
                     kb > 0 || kk > 0);
          tc_commit2_mc(&empty_bar[stage], 0x3);
          if (++stage == OG_STAGES) { stage = 0; phase ^= 1; }
        }
        if (!ok) break;
        tc_commit2_mc(&tfull_bar[acc], 0x3);
        if (++acc == 2) { acc = 0; acc_phase ^= 1; }
      }
      // the last products have completed before the CTAs leave
      if (--stage < 0) { stage = OG_STAGES - 1; phase ^= 1; }
      mbar_wait_poll(&empty_bar[stage], phase, nullptr, 0);
    }
  } else {
    const int q = warp & 3, part = (warp - 2) >> 2;
    uint8_t* out = smem + (OG_OUT + 1023) / 1024 * 1024 + (warp - 2) * 4 * OG_PIECE;
    int acc = 0, pieces = 0;
    uint32_t acc_phase = 0;
    const bool keep = !failed(p.status);
    const uint32_t leader_tempty = map_to_cta(smem_u32(&tempty_bar[0]), 0);
    for (int tile = cluster; tile < p.total; tile += clusters) {
      int cls, mat, ti, tj;
      ortho_tile<TILE>(p, tile, cls, mat, ti, tj);
      Addend add(p, mat, ti * TILE + crank * 128 + q * 32 + lane, tj * TILE + part * (TILE / 2));
      if (!__all_sync(0xffffffffu, own_poll(&tfull_bar[acc], acc_phase, p.status, ERR_TIMEOUT_TMEM_FULL))) break;
      tc_fence_after();
      ortho_epilogue<TILE / 2>(p, cls ? &maps.c[1] : &maps.c[0], out,
                               tmem_base + acc * TILE + part * (TILE / 2) + (static_cast<uint32_t>(q * 32) << 16),
                               mat + (cls ? p.cls[1].c0 : p.cls[0].c0), add, ti * TILE + crank * 128 + q * 32,
                               tj * TILE + part * (TILE / 2), cls ? p.cls[1].N : p.cls[0].N, keep, p.sym && ti != tj, lane, pieces);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_remote(leader_tempty + acc * 8);
      if (++acc == 2) { acc = 0; acc_phase ^= 1; }
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  tc_fence_after();
  if (warp == 1) tmem_dealloc2(tmem_base, 2 * TILE);
}

// S from the sums that several CTAs left for each tile on and below the diagonal, added up in order: 16 rows of a tile per block.
__global__ void __launch_bounds__(256) ortho_reduce_kernel(const float* __restrict__ partial, int splits, int tiles, int d,
                                                           __half* __restrict__ S, long long stride, int ld, float alpha) {
  chain_point();
  const int strip = blockIdx.x & 7, unit = blockIdx.x >> 3, mat = unit / tiles;
  OrthoGemm place{};
  place.sym = 1;
  place.cls[0].tiles = tiles;
  place.cls[0].count = mat + 1;
  int cls, m, ti, tj;
  ortho_tile<128>(place, unit, cls, m, ti, tj);
  const int r = strip * 16 + (threadIdx.x >> 4), c = (threadIdx.x & 15) * 8;
  const float4* from = reinterpret_cast<const float4*>(partial + static_cast<long long>(unit) * splits * (128 * 128) + r * 128 + c);
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
#pragma unroll 4
  for (int k = 0; k < splits; ++k) {
    const float4 a = from[k * (128 * 32)], b = from[k * (128 * 32) + 1];
    x.x += a.x; x.y += a.y; x.z += a.z; x.w += a.w;
    y.x += b.x; y.y += b.y; y.z += b.z; y.w += b.w;
  }
  const int row = ti * 128 + r, col = tj * 128 + c;
  if (row >= d || col >= ld) return;
  const __half2 h[4] = {__floats2half2_rn(alpha * x.x, alpha * x.y), __floats2half2_rn(alpha * x.z, alpha * x.w),
                        __floats2half2_rn(alpha * y.x, alpha * y.y), __floats2half2_rn(alpha * y.z, alpha * y.w)};
  S += mat * stride;
  *reinterpret_cast<uint4*>(S + static_cast<long long>(row) * ld + col) = *reinterpret_cast<const uint4*>(h);
  if (ti != tj) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (col + j < d) S[static_cast<long long>(col + j) * ld + row] = j & 1 ? __high2half(h[j / 2]) : __low2half(h[j / 2]);
  }
}

// ------------------------------------------------------------------------------------------------ small matrices
// Everything for one matrix in one CTA and one launch, where X fits next to its factors: d <= 128, K <= 384. Bound by latency:
// three products a step whose operands never leave shared memory (X in blocks of 64 columns of 128 swizzled rows, which serve
// as the K-major operands of X X^T and as the MN-major one of P X), accumulators in tensor memory, a barrier or two between.
// Eight matrices of 64 x 64: 64 us by the launches above, 33 of them on the host, 13 by this one.
constexpr int OS_MAX_D = 128, OS_MAX_K = 384, OS_THREADS = 512;
// Threads: a warp for 32 rows and 32 columns of a square factor, 16 warps above 64 rows and 8 up to there (eight 128 x 384 by 8 warps
// 42.7 us, by 16 38; 64 x 64 12.2 and 13.2).
constexpr int os_threads(int d) { return d > 64 ? OS_THREADS : OS_THREADS / 2; }
constexpr int OS_BLOCK = 128 * 128;           // 64 columns of 128 rows, in bytes
constexpr int OS_S = (OS_MAX_K / 64) * OS_BLOCK, OS_P = OS_S + 2 * OS_BLOCK, OS_BARS = OS_P + 2 * OS_BLOCK;
constexpr int OS_SMEM = OS_BARS + 256 + 1024;

__device__ __forceinline__ uint32_t os_at(int row, int col) {         // byte offset of an element of X, S or P
  return (col >> 6) * OS_BLOCK + row * 128 + ((((col & 63) >> 3) ^ (row & 7)) << 4) + (col & 7) * 2;
}
// 32 values of one row from column `col` (a multiple of 32) on, scaled and rounded
__device__ __forceinline__ void os_put(uint8_t* to, int row, int col, const float (&f)[32]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const __half2 h = __floats2half2_rn(f[8 * i + 2 * j], f[8 * i + 2 * j + 1]);
      w[j] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(to + os_at(row, col + 8 * i)) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

template <bool STEP>
__global__ void __launch_bounds__(OS_THREADS, 1)
ortho_small_kernel(const OrthoGroups a, const OrthoInput in, const OrthoGroups b, const OrthoOutput o, double eps, int steps) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + OS_BARS);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar + 1);
  double* red = reinterpret_cast<double*>(bar + 4);
  int* gave_up = reinterpret_cast<int*>(bar + 4 + OS_THREADS / 32);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, threads = blockDim.x;
  if (threadIdx.x == 0) {
    mbar_init(bar, 1);
    fence_barrier_init();
    *gave_up = 0;
  }
  if (warp == 0) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  chain_point();

  const OrthoPlace p = ortho_place(a);
  if (STEP && warp == 1) ortho_apart(a, p);
  const OrthoGroup& m = a.g[p.group];
  const bool upright = m.rows > m.cols;
  const int d = upright ? m.cols : m.rows, K = upright ? m.rows : m.cols;
  const int blocks = (K + 63) / 64;
  for (int i = threadIdx.x; i < blocks * OS_BLOCK / 16; i += threads) reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
  const float gs = STEP ? step_scale(in) : 0.f;
  double sum = 0;
  // The matrix in vectors of W = 4 elements or 1, four per thread at a time: `before` for all four (loads), then `work`, both
  // with (row, column, address, number of the four). Element by element the three passes took 41 of 64 us of a 128 x 384.
  constexpr int U = 4;
  auto walk = [&](auto width, int ld, long long at, auto before, auto work) {
    constexpr int W = decltype(width)::value;
    const int per_row = m.cols / W, down = threads / per_row, over = threads - down * per_row;
    int r = threadIdx.x / per_row, c = threadIdx.x - r * per_row;
    while (r < m.rows) {
      int rr[U], cc[U];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        rr[k] = r;
        cc[k] = c * W;
        r += down;
        c += over;
        if (c >= per_row) c -= per_row, ++r;
        if (rr[k] < m.rows) before(rr[k], cc[k], at + static_cast<long long>(rr[k]) * ld + cc[k], k);
      }
#pragma unroll
      for (int k = 0; k < U; ++k)
        if (rr[k] < m.rows) work(rr[k], cc[k], at + static_cast<long long>(rr[k]) * ld + cc[k], k);
    }
  };
  auto at_width = [&](bool four, auto f) {
    if (four) f(std::integral_constant<int, 4>{});
    else f(std::integral_constant<int, 1>{});
  };
  float4 x[U], y[U];                          // .x alone where the width is 1
  auto load = [&](auto width) {
    return [&](int, int, long long e, int k) {
      if (decltype(width)::value == 4) {
        x[k] = STEP ? *reinterpret_cast<const float4*>(in.grad + e) : in_value4(in, e);
        if (STEP) y[k] = *reinterpret_cast<const float4*>(in.momentum + e);
      } else {
        x[k] = make_float4(STEP ? in.grad[e] : in_value(in, e), 0.f, 0.f, 0.f);
        y[k] = make_float4(STEP ? in.momentum[e] : 0.f, 0.f, 0.f, 0.f);
      }
    };
  };
  auto moved = [&](float g, float& mom) {
    g = clean(g * gs);
    mom = in.beta * mom + (1.f - in.beta) * g;
    return in.nesterov ? in.beta * mom + (1.f - in.beta) * g : mom;
  };
  if (p.found)
    at_width(p.four, [&](auto width) {
      walk(width, m.ld, p.at, load(width), [&](int, int, long long e, int k) {
        if (STEP) {
          x[k] = make_float4(moved(x[k].x, y[k].x), moved(x[k].y, y[k].y), moved(x[k].z, y[k].z), moved(x[k].w, y[k].w));
          if (decltype(width)::value == 4) *reinterpret_cast<float4*>(in.momentum + e) = y[k];
          else in.momentum[e] = y[k].x, x[k].y = x[k].z = x[k].w = 0.f;
        }
        const float4 u[1] = {x[k]};
        sum += squares_of(u);
      });
    });
  for (int k = 16; k > 0; k >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
  if (lane == 0) red[warp] = sum;
  __syncthreads();
  sum = 0;
  for (int i = 0; i < threads / 32; ++i) sum += red[i];
  const double norm = sqrt(sum);
  const NormScale scale(norm, eps);
  if (p.found)                                // each thread reads what it has written
    at_width(p.four, [&](auto width) {
      constexpr int W = decltype(width)::value;
      walk(width, m.ld, p.at, load(width), [&](int r, int c, long long e, int k) {
        float u[4] = {x[k].x, x[k].y, x[k].z, x[k].w};
        const float mom[4] = {y[k].x, y[k].y, y[k].z, y[k].w};
        if (STEP) {
#pragma unroll
          for (int j = 0; j < W; ++j) {
            const float g = clean(u[j] * gs);
            u[j] = in.nesterov ? in.beta * mom[j] + (1.f - in.beta) * g : mom[j];
          }
          if (in.zero_grad) {
            if (W == 4) *reinterpret_cast<float4*>(in.grad + e) = make_float4(0.f, 0.f, 0.f, 0.f);
            else in.grad[e] = 0.f;
          }
        }
        if (W == 4 && !upright) {
          const __half2 h[2] = {__floats2half2_rn(scale(u[0]), scale(u[1])), __floats2half2_rn(scale(u[2]), scale(u[3]))};
          *reinterpret_cast<uint2*>(smem + os_at(r, c)) = *reinterpret_cast<const uint2*>(h);
        } else {
#pragma unroll
          for (int j = 0; j < W; ++j)
            *reinterpret_cast<__half*>(smem + (upright ? os_at(c + j, r) : os_at(r, c + j))) = __float2half_rn(scale(u[j]));
        }
      });
    });

  const int q = warp & 3, part = warp >> 2, row = q * 32 + lane;
  const uint32_t lanes = static_cast<uint32_t>(q * 32) << 16, t_s = tmem + OS_MAX_K;
  const uint32_t x_at = smem_u32(smem), s_at = smem_u32(smem + OS_S), p_at = smem_u32(smem + OS_P);
  const int wide = d > 64 ? 128 : 64;         // columns of the square factors
  uint32_t phase = 0;
  bool ok = true;
  const uint32_t lead = lane == 0;
  // all threads: what they wrote to shared memory is there for the products, which warp 0 issues and all wait for
  auto products = [&](auto issue) {
    fence_proxy_async_smem();
    tc_fence_before();
    __syncthreads();
    if (!ok) return;                          // with this warp's last products perhaps still under way
    if (warp == 0) {
      tc_fence_after();
      issue();
      tc_commit_warp(lead, smem_u32(bar));
    }
    ok = mbar_wait_warp(bar, phase, a.status, ERR_TIMEOUT_TMEM_FULL);
    if (ok) phase ^= 1;
    else *gave_up = 1;
    tc_fence_after();
  };
  for (int step = 0; step < steps; ++step) {
    products([&] {
      for (int k = 0; k < blocks; ++k) {
        const uint32_t lo = smem_desc_lo(x_at + k * OS_BLOCK, 0);
        umma_ss4_warp<2, 2>(lead, t_s, lo, lo, make_idesc_fp16(128, wide, 0), k > 0);
      }
    });
    float s[32];
    const int c0 = part * 32;                 // this warp's columns of the factors
    if (c0 < wide) {
      uint32_t v[32];
      tmem_ld32(t_s + lanes + c0, v);
      tmem_wait_ld();
#pragma unroll
      for (int j = 0; j < 32; ++j)           // b S takes S as it is in c S^2: near 1 most of a rounding cancels between the two
        s[j] = __half2float(__float2half_rn(__uint_as_float(v[j]) * (1.f / NS_SCALE)));
      os_put(smem + OS_S, row, c0, s);
    }
    products([&] {
      for (int k = 0; k < wide / 64; ++k) {
        const uint32_t lo = smem_desc_lo(s_at + k * OS_BLOCK, 0);
        umma_ss4_warp<2, 2>(lead, t_s, lo, lo, make_idesc_fp16(128, wide, 0), k > 0);
      }
    });
    if (c0 < wide) {
      uint32_t v[32];
      tmem_ld32(t_s + lanes + c0, v);
      tmem_wait_ld();
      float f[32];
#pragma unroll
      for (int j = 0; j < 32; ++j)
        f[j] = NS_C / NS_SCALE * __uint_as_float(v[j]) + NS_B * s[j] + (row == c0 + j ? NS_A * NS_SCALE : 0.f);
      os_put(smem + OS_P, row, c0, f);
    }
    products([&] {
      for (int c = 0; c < blocks * 64; c += 256) {
        const int cols = min(256, blocks * 64 - c);
        for (int k = 0; k < wide / 64; ++k)
          umma_ss4_warp<2, 128>(lead, tmem + c, smem_desc_lo(p_at + k * OS_BLOCK, 0),
                                smem_desc_lo(x_at + (c >> 6) * OS_BLOCK + k * 8192, OS_BLOCK), make_idesc_fp16(128, cols, 1), k > 0);
      }
    });
    for (int c = part * 32; c < blocks * 64; c += threads / 4) {
      uint32_t v[32];
      tmem_ld32(tmem + lanes + c, v);
      tmem_wait_ld();
      float f[32];
#pragma unroll
      for (int j = 0; j < 32; ++j) f[j] = __uint_as_float(v[j]) * (1.f / NS_SCALE);
      os_put(smem, row, c, f);
    }
  }
  if (warp == 0 && !ok) mbar_wait_warp(bar, phase, nullptr, 0);       // the last products, before the tensor memory goes back
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) tmem_dealloc(tmem, 512);
  const OrthoGroup& t = b.g[p.group];
  if (!p.found || *gave_up || failed(a.status)) return;
  const long long out_at = t.offsets ? p.at : p.matrix * t.stride;
  const bool average = STEP && o.ema && o.ema_beta >= 0.f;
  const bool four = b.aligned && t.cols % 4 == 0 && t.ld % 4 == 0 && out_at % 4 == 0;
  at_width(four, [&](auto width) {
    constexpr int W = decltype(width)::value;
    walk(
        width, t.ld, out_at,
        [&](int, int, long long e, int k) {
          if (W == 4) {
            if (STEP) x[k] = *reinterpret_cast<const float4*>(o.master + e);
            if (average) y[k] = *reinterpret_cast<const float4*>(o.ema + e);
          } else {
            if (STEP) x[k].x = o.master[e];
            if (average) y[k].x = o.ema[e];
          }
        },
        [&](int r, int c, long long e, int k) {
          float v[4];
          const float old[4] = {x[k].x, x[k].y, x[k].z, x[k].w}, mean[4] = {y[k].x, y[k].y, y[k].z, y[k].w};
#pragma unroll
          for (int j = 0; j < W; ++j) {
            v[j] = __half2float(*reinterpret_cast<const __half*>(smem + (upright ? os_at(c + j, r) : os_at(r, c + j)))) * (1.f / NS_SCALE);
            if (STEP) v[j] = old[j] * o.decay - m.rate * v[j];
          }
          if (W == 4) {
            const uint2 low = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
            if (!STEP) *reinterpret_cast<uint2*>(o.out + e) = low;
            if (STEP) *reinterpret_cast<float4*>(o.master + e) = make_float4(v[0], v[1], v[2], v[3]);
            if (STEP && o.weights) *reinterpret_cast<uint2*>(o.weights + e) = low;
            if (average)
              *reinterpret_cast<float4*>(o.ema + e) =
                  make_float4(v[0] + o.ema_beta * (mean[0] - v[0]), v[1] + o.ema_beta * (mean[1] - v[1]),
                              v[2] + o.ema_beta * (mean[2] - v[2]), v[3] + o.ema_beta * (mean[3] - v[3]));
          } else {
            if (!STEP) o.out[e] = __float2bfloat16_rn(v[0]);
            if (STEP) o.master[e] = v[0];
            if (STEP && o.weights) o.weights[e] = __float2bfloat16_rn(v[0]);
            if (average) o.ema[e] = v[0] + o.ema_beta * (mean[0] - v[0]);
          }
        });
  });
}

// ------------------------------------------------------------------------------------------------ few rows, long ones
// d <= 128 and longer rows: all steps on the Gram matrix alone, one CTA a matrix, and X is read twice instead of ten times. What
// keeps groups of steps from being longer than two elsewhere, the Gram matrix's rounding, is answered by precision here: sums of
// X X^T stay in 32 bits, and the [d, d] factors are kept as two fp16 numbers (22 bits), which a product takes as three. Their
// product Q is applied in both parts too: its entries reach a^5, and rounded to 11 bits they would leave 0.1 of a large direction.
// Bound by the chain of products, three deep a step and each three times over: 128 x 4000 takes 64 us in six launches (71 with 8
// warps here instead of 16), 64 x 4000 43.
constexpr float NS_Q_SCALE = 64.f;
constexpr int OL_MAX_STEPS = 5;               // a^5 times the scale is inside fp16's range
constexpr int OL_S = 0, OL_P = 4 * OS_BLOCK, OL_Q = 8 * OS_BLOCK, OL_BARS = 12 * OS_BLOCK;      // hi, then lo
constexpr int OL_SMEM = OL_BARS + 256 + 1024;
constexpr int OL_MAX_SPLITS = 12;

__device__ __forceinline__ void split_half(const float (&f)[32], float (&lo)[32]) {
#pragma unroll
  for (int j = 0; j < 32; ++j) lo[j] = f[j] - __half2float(__float2half_rn(f[j]));
}
__device__ __forceinline__ void os_put2(uint8_t* to, int row, int col, const float (&f)[32]) {
  float lo[32];
  split_half(f, lo);
  os_put(to, row, col, f);
  os_put(to + 2 * OS_BLOCK, row, col, lo);
}

// `partial`: [matrix, split, 128, 128] sums of X X^T; Q: [2, count] matrices of d rows of pitch ld (hi, lo).
__global__ void __launch_bounds__(OS_THREADS, 1)
ortho_polynomial_kernel(const float* __restrict__ partial, int splits, __half* __restrict__ Q, int count, int d, int ld, int steps,
                        int* status) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + OL_BARS);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(bar, 1);
    fence_barrier_init();
  }
  if (warp == 0) {
    tmem_alloc(tmem_slot, 256);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  chain_point();

  const int q = warp & 3, part = warp >> 2, row = q * 32 + lane;
  const int wide = d > 64 ? 128 : 64, c0 = part * 32;        // this warp's columns
  const bool mine = c0 < wide;
  const uint32_t lanes = static_cast<uint32_t>(q * 32) << 16;
  uint8_t *S = smem + OL_S, *P = smem + OL_P, *QQ = smem + OL_Q;
  uint32_t phase = 0;
  auto begin = [&] {
    fence_proxy_async_smem();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
  };
  const uint32_t lead = lane == 0;
  auto product = [&](uint32_t to, const uint8_t* a, const uint8_t* b) {        // warp 0; small terms first
    const uint32_t a_hi = smem_desc_lo(smem_u32(a), 0), b_hi = smem_desc_lo(smem_u32(b), 0);
    constexpr uint32_t BLOCK = OS_BLOCK / 16, LO = 2 * BLOCK;
    const uint32_t idesc = make_idesc_fp16(128, wide, 0);
    for (int k = 0; k < wide / 64; ++k) umma_ss4_warp<2, 2>(lead, tmem + to, a_hi + LO + k * BLOCK, b_hi + k * BLOCK, idesc, k > 0);
    for (int k = 0; k < wide / 64; ++k) umma_ss4_warp<2, 2>(lead, tmem + to, a_hi + k * BLOCK, b_hi + LO + k * BLOCK, idesc, 1);
    for (int k = 0; k < wide / 64; ++k) umma_ss4_warp<2, 2>(lead, tmem + to, a_hi + k * BLOCK, b_hi + k * BLOCK, idesc, 1);
  };
  bool ok = true;
  auto finish = [&] {
    if (!ok) return;                          // with warp 0's last products perhaps still under way
    if (warp == 0) tc_commit_warp(lead, smem_u32(bar));
    ok = mbar_wait_warp(bar, phase, status, ERR_TIMEOUT_TMEM_FULL);
    if (ok) phase ^= 1;
    tc_fence_after();
  };
  // the sums, side by side through the (still free) place of Q, whose 16-byte chunks are swizzled by row
  float4* sums = reinterpret_cast<float4*>(QQ);
  const float4* from = reinterpret_cast<const float4*>(partial) + static_cast<long long>(blockIdx.x) * splits * (128 * 32);
  for (int i = threadIdx.x; i < wide * (wide / 4); i += OS_THREADS) {
    const int r = i / (wide / 4), c = i % (wide / 4);
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int k = 0; k < splits; ++k) {
      const float4 y = from[k * (128 * 32) + r * 32 + c];
      x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
    }
    sums[r * 32 + (c ^ (r & 7))] = x;
  }
  __syncthreads();
  float s[32];
  if (mine) {
    float f[32];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float4 x = row < wide ? sums[row * 32 + ((c0 / 4 + j) ^ (row & 7))] : make_float4(0.f, 0.f, 0.f, 0.f);
      f[4 * j] = x.x; f[4 * j + 1] = x.y; f[4 * j + 2] = x.z; f[4 * j + 3] = x.w;
    }
#pragma unroll
    for (int j = 0; j < 32; ++j) s[j] = f[j] *= 1.f / NS_SCALE;
    os_put2(S, row, c0, f);
  }
  __syncthreads();                            // all sums are taken before Q comes
  // this lane's columns c0 + 32 h .. of an accumulator, times alpha
  auto take = [&](uint32_t from, float alpha, float (&f)[32]) {
    uint32_t v[32];
    tmem_ld32(tmem + from + lanes + c0, v);
    tmem_wait_ld();
#pragma unroll
    for (int j = 0; j < 32; ++j) f[j] = alpha * __uint_as_float(v[j]);
  };
  for (int step = 0; step < steps; ++step) {
    const bool last = step + 1 == steps;
    begin();
    if (warp == 0 && ok) product(0, S, S);
    finish();
    if (mine) {
      float f[32];
      take(0, NS_C / NS_SCALE, f);
#pragma unroll
      for (int j = 0; j < 32; ++j) f[j] += NS_B * s[j] + (row == c0 + j ? NS_A * NS_SCALE : 0.f);
      os_put2(P, row, c0, f);
      if (step == 0) {
#pragma unroll
        for (int j = 0; j < 32; ++j) f[j] *= NS_Q_SCALE / NS_SCALE;
        os_put2(QQ, row, c0, f);
      }
    }
    if (step || !last) {
      begin();
      if (warp == 0 && ok) {
        if (step) product(128, P, QQ);
        if (!last) product(0, P, S);
      }
      finish();
    }
    if (mine) {
      float f[32];
      if (step) {
        take(128, 1.f / NS_SCALE, f);
        os_put2(QQ, row, c0, f);
      }
      if (!last) {
        take(0, 1.f / NS_SCALE, f);
        os_put2(S, row, c0, f);      // P S takes the place of S
      }
    }
    if (last) break;
    begin();
    if (warp == 0 && ok) product(0, S, P);
    finish();
    if (mine) {
      float f[32];
      take(0, 1.f / NS_SCALE, f);
#pragma unroll
      for (int j = 0; j < 32; ++j) s[j] = f[j];
      os_put2(S, row, c0, f);
    }
  }
  if (warp == 0 && !ok) mbar_wait_warp(bar, phase, nullptr, 0);       // the last products, before the tensor memory goes back
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) tmem_dealloc(tmem, 256);
  __half* to = Q + static_cast<long long>(blockIdx.x) * d * ld;
  const long long low = static_cast<long long>(count) * d * ld;
  for (int i = threadIdx.x; i < d * (wide / 8); i += OS_THREADS) {
    const int r = i / (wide / 8), c = i % (wide / 8) * 8;
    if (c >= ld) continue;
    *reinterpret_cast<uint4*>(to + r * ld + c) = *reinterpret_cast<const uint4*>(QQ + os_at(r, c));
    *reinterpret_cast<uint4*>(to + low + r * ld + c) = *reinterpret_cast<const uint4*>(QQ + 2 * OS_BLOCK + os_at(r, c));
  }
}

// ------------------------------------------------------------------------------------------------ host side
namespace {

// Lets a kernel have `bytes` of shared memory, once a device.
template <typename F> bool allow_smem(F kernel, int bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  const uint64_t bit = 1ull << (dev & 63);
  if (done.load(std::memory_order_relaxed) & bit) return true;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
  done.fetch_or(bit, std::memory_order_relaxed);
  return true;
}

int pitch(int n) { return (n + 63) / 64 * 64; }
bool on_grid(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// How the steps are grouped. One step by itself is a Gram matrix of X, its square and an update of X: in units of d^3, with
// symmetric products at half and r = K / d, 3 r + 1. Two steps can share the update: the Gram matrix alone goes on (S <- P S P
// with P = a I + b S + c S^2, all symmetric and commuting) and X is multiplied by the product of both P at the end: 3 r + 5
// instead of 6 r + 2, the less for every oblong matrix. But a Gram matrix's rounding error (2^-12 of its norm) grows by a^2 a step
// in directions that hold little of the norm, and is not small against them any more. So pairs of steps alternate with single
// ones: error on 333 x 1001 gradients with half as much noise as signal 1.13e-3 by single steps, 1.09e-3 as 2, 1, 2, 1.49e-3 as
// 2, 2, 1, 1.8e-3 as 3, 2; on 127 x 640 6e-4, 6e-4, 6e-4, 1.8e-3; a group of five diverges. Below GROUP_FROM rows single steps:
// the products are no longer than their launches, of which groups have two more (us by single steps / in pairs: 256 x 600 94 / 101,
// ten 333 x 1001 139 / 142, 42 of 384 x 1024 282 / 266, 30 of 500 x 1500 434 / 397), and a handful of rows does not average the
// roundings (5 x 9: up to three times the error of single steps). K is the longest side of the batch: square matrices beside oblong
// ones go in pairs with them, which costs them nothing (4 d^3 a step either way).
constexpr int GROUP_FROM = 384;
struct Groups {
  int n, size[20];
};
Groups groups_of(int d, int K, int steps) {
  Groups g = {0, {}};
  for (int left = steps; left > 0; left -= g.size[g.n++]) g.size[g.n] = K > d && d >= GROUP_FROM && left > 1 && g.n % 2 == 0 ? 2 : 1;
  return g;
}
int buffers_of(const Groups& g) { return g.size[0] == 1 ? 2 : 4; }

enum Factor { F_S, F_P0, F_T, F_P1 };         // where the [d, d] factors of a batch are

// Workspace of a batch: partial sums, both X of every class, the factors.
struct Layout {
  int d, count, classes, K[NS_CLASSES], members[NS_CLASSES], group_class[NS_GROUPS], group_first[NS_GROUPS];
  Groups steps;
  bool few;                                   // all steps on the Gram matrix
  long long x_at[NS_CLASSES], s_at, partial_at, bytes;
  long long x_stride(int c) const { return static_cast<long long>(d) * pitch(K[c]); }
  long long s_stride() const { return static_cast<long long>(d) * pitch(d); }
  int fill(const AerisOrtho& a);
};
bool small(const Layout& l) { return l.d <= OS_MAX_D && l.K[0] <= OS_MAX_K; }
// CTAs that share one matrix's X X^T where rows are few: eight blocks of 64 each, up to OL_MAX_SPLITS. By the length alone: with few
// rows a matrix has the same bits in every batch.
int splits_of(const Layout& l, int c) {
  const int blocks = (l.K[c] + OG_BK - 1) / OG_BK, s = blocks / 8 < OL_MAX_SPLITS ? blocks / 8 : OL_MAX_SPLITS;
  if (s < 2) return 1;
  const int each = (blocks + s - 1) / s;
  return (blocks + each - 1) / each;          // none of them empty
}
// The same for X X^T of longer sides whose tiles leave most of the GPU idle: seven 151 x 4472 have 21 tiles of 70 blocks, 16 us by
// themselves and 4 in parts, plus 4 for adding those up. 1: in one piece. By how many matrices there are too: a sum's order, and with it
// its last bits, is another alone and among seven.
int gram_splits(const Layout& l) {
  if (l.few || l.classes > 1) return 1;
  const int m = (l.d + 127) / 128, blocks = (l.K[0] + OG_BK - 1) / OG_BK;
  const long long units = static_cast<long long>(m) * (m + 1) / 2 * l.count;
  if (2 * units > num_sms()) return 1;
  int s = num_sms() / static_cast<int>(units);
  if (s > blocks / 6) s = blocks / 6;
  if (s < 2) return 1;
  const int each = (blocks + s - 1) / s;
  return (blocks - each) * 0.235 > 6 ? (blocks + each - 1) / each : 1;
}
int Layout::fill(const AerisOrtho& a) {
  if (a.groups < 1 || a.groups > NS_GROUPS || a.steps < 1 || a.steps > 20) return -1;
  d = count = classes = 0;
  for (int i = 0; i < a.groups; ++i) {
    const AerisOrthoGroup& g = a.group[i];
    if (g.rows < 1 || g.cols < 1 || g.count < 1 || g.count > (1 << 20) || g.ld < g.cols) return -2;
    const int shorter = g.rows < g.cols ? g.rows : g.cols, longer = g.rows < g.cols ? g.cols : g.rows;
    if (longer > NS_MAX_SIDE) return -2;
    if (i && shorter != d) return -3;
    d = shorter;
    int c = 0;
    while (c < classes && K[c] != longer) ++c;
    if (c == NS_CLASSES) return -4;
    if (c == classes) K[classes] = longer, members[classes++] = 0;
    group_class[i] = c;
    group_first[i] = members[c];
    members[c] += g.count;
    count += g.count;
  }
  if (classes == 2 && K[0] < K[1]) {          // the longer tiles first: they leave the shorter tail
    int t = K[0];
    K[0] = K[1], K[1] = t, t = members[0], members[0] = members[1], members[1] = t;
    for (int i = 0; i < a.groups; ++i) group_class[i] ^= 1;
  }
  bytes = 0;
  few = false;
  if (small(*this)) return 0;                 // everything in shared memory
  few = d <= OS_MAX_D && a.steps <= OL_MAX_STEPS;
  steps = groups_of(d, K[0], a.steps);
  bytes = (static_cast<long long>(count) * NS_PARTS * 8 + 1023) / 1024 * 1024;
  for (int c = 0; c < classes; ++c) {
    x_at[c] = bytes;
    bytes += (2ll * members[c] * x_stride(c) * 2 + 1023) / 1024 * 1024;
  }
  s_at = bytes;
  bytes += (static_cast<long long>(few ? 2 : buffers_of(steps)) * count * s_stride() * 2 + 1023) / 1024 * 1024;
  partial_at = bytes;
  if (few) {
    if (classes > 1) return -10;
    bytes += static_cast<long long>(splits_of(*this, 0)) * count * (128 * 128 * 4);
  } else if (const int splits = gram_splits(*this); splits > 1) {
    const int m = (d + 127) / 128;
    bytes += static_cast<long long>(splits) * count * (m * (m + 1) / 2) * (128 * 128 * 4);
  }
  return 0;
}

// The products of a batch by their sizes: S = X X^T, factor times factor, factor times X.
OrthoGemm empty_gemm() {
  OrthoGemm p{};
  for (int c = 0; c < NS_CLASSES; ++c) p.cls[c].N = p.cls[c].K = 1;        // a class without matrices
  p.alpha = 1.f / NS_SCALE;
  return p;
}
OrthoGemm gram_gemm(const Layout& l) {
  OrthoGemm p = empty_gemm();
  p.sym = 1;
  p.M = l.d;
  for (int c = 0; c < l.classes; ++c) p.cls[c].count = l.members[c], p.cls[c].N = l.d, p.cls[c].K = l.K[c];
  return p;
}
OrthoGemm factor_gemm(const Layout& l) {
  OrthoGemm p = empty_gemm();
  p.sym = 1;
  p.M = l.d;
  p.cls[0].count = l.count;
  p.cls[0].N = p.cls[0].K = l.d;
  return p;
}
OrthoGemm update_gemm(const Layout& l) {
  OrthoGemm p = empty_gemm();
  p.M = l.d;
  for (int c = 0; c < l.classes; ++c) p.cls[c].count = l.members[c], p.cls[c].N = l.K[c], p.cls[c].K = l.d;
  return p;
}
long long tiles_of(const OrthoGemm& p, int c, int tile) {
  const long long m = (p.M + tile - 1) / tile, n = (p.cls[c].N + tile - 1) / tile;
  return p.sym ? m * (m + 1) / 2 : m * n;
}
// us of a launch: a start and an end, and for every round of tiles a fixed part and one per block of 64 of the reduction (the
// mean over both classes). Measured, single / pair: 10 x 333 rows and columns over 384 8.2 / 11.0, 8 x (512 x 2048 over 512)
// 15.6 / 14.9, 6 x (1024 x 4096 over 1024) 53.7 / 43.5, 16 x 1536 over 1536 68.7 / 58.3, 2 x 1536 over 4096 37.1 / 31.0.
double cost_of(const OrthoGemm& p, int tile, int units, double ends, double round, double block) {
  long long total = 0, blocks = 0;
  for (int c = 0; c < NS_CLASSES; ++c) {
    const long long n = tiles_of(p, c, tile) * p.cls[c].count;
    total += n;
    blocks += n * ((p.cls[c].K + OG_BK - 1) / OG_BK);
  }
  return ends + static_cast<double>((total + units - 1) / units) * (round + block * blocks / total);
}
bool takes_pairs(const OrthoGemm& p) {
  return cost_of(p, 256, num_sms() / 2, 7, 1.6, 0.36) < cost_of(p, 128, num_sms(), 4.5, 1.3, 0.235);
}

struct Products {
  const Layout& l;
  __half* S;
  float* partial;
  __half* X[NS_CLASSES];
  CUtensorMap load_x[NS_CLASSES], store_x[NS_CLASSES], load_s, store_s;
  int* status;
  cudaStream_t stream;
  int launches = 0, rc = 0;

  Products(const Layout& layout, char* work, int* status_, cudaStream_t stream_) : l(layout), status(status_), stream(stream_) {
    S = reinterpret_cast<__half*>(work + l.s_at);
    partial = reinterpret_cast<float*>(work + l.partial_at);
    const uint64_t factors = static_cast<uint64_t>(l.few ? 2 : buffers_of(l.steps)) * l.count;
    rc = make_tmap_3d_fp16(&load_s, S, l.d, l.d, factors, pitch(l.d), 64, 64);
    if (!rc) rc = make_tmap_3d_fp16(&store_s, S, l.d, l.d, factors, pitch(l.d), 32, 32);
    for (int c = 0; c < l.classes; ++c) {
      X[c] = reinterpret_cast<__half*>(work + l.x_at[c]);
      if (!rc) rc = make_tmap_3d_fp16(&load_x[c], X[c], l.K[c], l.d, 2ull * l.members[c], pitch(l.K[c]), 64, 64);
      if (!rc) rc = make_tmap_3d_fp16(&store_x[c], X[c], l.K[c], l.d, 2ull * l.members[c], pitch(l.K[c]), 32, 32);
    }
  }
  template <int B_MN> void launch(const OrthoMaps& maps, OrthoGemm& p) {
    if (rc) return;
    p.status = status;
    const bool parts = p.partial || p.cls[0].low;
    const bool pair = !parts && takes_pairs(p);
    const int tile = pair ? 256 : 128, units = pair ? num_sms() / 2 : num_sms();
    long long total = 0;
    for (int c = 0; c < NS_CLASSES; ++c) total += tiles_of(p, c, tile) * p.cls[c].count;
    if (total > 0x7fffffff) {
      rc = -5;
      return;
    }
    for (int c = 0; c < NS_CLASSES; ++c) p.cls[c].tiles = static_cast<int>(tiles_of(p, c, tile));
    p.total = static_cast<int>(total) * (p.cls[0].splits > 1 ? p.cls[0].splits : 1);
    const int grid = (p.total < units ? p.total : units) * (pair ? 2 : 1);
    auto kern = pair ? ortho_gemm_pair_kernel<B_MN> : parts ? ortho_gemm_kernel<B_MN, true> : ortho_gemm_kernel<B_MN, false>;
    static std::atomic<uint64_t> done[3];
    rc = allow_smem(kern, OG_SMEM, done[pair ? 2 : parts]) ? launch_chained(kern, grid, OG_THREADS, OG_SMEM, stream, maps, p) : -20;
    ++launches;
  }
  OrthoMaps square() const {
    OrthoMaps m;
    m.a[0] = m.a[1] = m.b[0] = m.b[1] = load_s;
    m.c[0] = m.c[1] = store_s;
    return m;
  }
  OrthoGemm factors(int out, int i, int j) const {
    OrthoGemm p = factor_gemm(l);
    p.cls[0].a0 = i * l.count;
    p.cls[0].b0 = j * l.count;
    p.cls[0].c0 = out * l.count;
    return p;
  }
  void product(int out, int i, int j) {       // factor `out` = (factor i) (factor j)
    OrthoGemm p = factors(out, i, j);
    launch<0>(square(), p);
  }
  void polynomial(int out) {                  // factor `out` = a I + b S + c S^2
    OrthoGemm p = factors(out, F_S, F_S);
    p.R = S + F_S * l.count * l.s_stride();
    p.r_stride = l.s_stride();
    p.ldr = pitch(l.d);
    p.alpha = NS_C / NS_SCALE;
    p.beta = NS_B;
    p.gamma = NS_A * NS_SCALE;
    launch<0>(square(), p);
  }
  void gram(int from) {                       // S = X X^T
    OrthoGemm p = gram_gemm(l);
    OrthoMaps m = square();
    for (int c = 0, first = 0; c < l.classes; first += l.members[c++]) {
      m.a[c] = m.b[c] = load_x[c];
      p.cls[c].a0 = p.cls[c].b0 = from * l.members[c];
      p.cls[c].c0 = F_S * l.count + first;
    }
    const int splits = gram_splits(l);
    if (splits > 1) {
      p.cls[0].splits = splits;
      p.partial = partial;
    }
    launch<0>(m, p);
    if (splits == 1 || rc) return;
    const int units = p.cls[0].tiles * l.count;
    rc = launch_chained(ortho_reduce_kernel, units * 8, 256, 0, stream, static_cast<const float*>(partial), splits, p.cls[0].tiles, l.d,
                        at(F_S), l.s_stride(), pitch(l.d), 1.f / NS_SCALE);
    ++launches;
  }
  void update(int from, int by) {             // the other X = factor `by` X
    OrthoGemm p = update_gemm(l);
    OrthoMaps m = square();
    for (int c = 0, first = 0; c < l.classes; first += l.members[c++]) {
      m.b[c] = load_x[c];
      m.c[c] = store_x[c];
      p.cls[c].a0 = by * l.count + first;
      p.cls[c].b0 = from * l.members[c];
      p.cls[c].c0 = (1 - from) * l.members[c];
    }
    launch<1>(m, p);
  }
  // all steps on X number 0, into the other one
  __half* at(int f) const { return S + static_cast<long long>(f) * l.count * l.s_stride(); }
  void few(int splits, int steps) {
    OrthoGemm g = gram_gemm(l);
    OrthoMaps m = square();
    m.a[0] = m.b[0] = load_x[0];
    g.cls[0].splits = splits;
    g.partial = partial;
    launch<0>(m, g);
    if (rc) return;
    static std::atomic<uint64_t> done;
    if (!allow_smem(ortho_polynomial_kernel, OL_SMEM, done)) {
      rc = -20;
      return;
    }
    rc = launch_chained(ortho_polynomial_kernel, l.count, OS_THREADS, OL_SMEM, stream, static_cast<const float*>(partial), splits, S,
                        l.count, l.d, pitch(l.d), steps, status);
    ++launches;
    OrthoGemm u = update_gemm(l);
    m = square();
    m.b[0] = load_x[0];
    m.c[0] = store_x[0];
    u.cls[0].low = l.count;
    u.cls[0].c0 = l.count;
    u.alpha = 1.f / NS_Q_SCALE;
    launch<1>(m, u);
  }
  void group(int from, int steps) {           // one or two steps on X number `from`, into the other one
    gram(from);
    polynomial(F_P0);
    if (steps == 1) return update(from, F_P0);
    product(F_T, F_P0, F_S);
    product(F_S, F_T, F_P0);                  // S after the first step
    polynomial(F_P1);
    product(F_T, F_P1, F_P0);
    update(from, F_T);
  }
};

}  // namespace
}  // namespace aeris

using namespace aeris;

extern "C" long long aeris_ortho_work_bytes(const AerisOrtho* a) {
  Layout l;
  const int rc = l.fill(*a);
  return rc ? rc : l.bytes;
}

extern "C" int aeris_ortho_route(const AerisOrtho* a) {
  Layout l;
  if (const int rc = l.fill(*a)) return rc;
  if (small(l)) return ORTHO_ROUTE_ONE_LAUNCH;
  if (l.few) return ORTHO_ROUTE_GRAM_ALONE;
  const bool parts = gram_splits(l) > 1;
  return (l.steps.size[0] == 2 ? ORTHO_ROUTE_TWO_STEPS : 0) | (parts ? ORTHO_ROUTE_GRAM_PARTS : 0) |
         (!parts && takes_pairs(gram_gemm(l)) ? ORTHO_ROUTE_GRAM_PAIRS : 0) |
         (takes_pairs(factor_gemm(l)) ? ORTHO_ROUTE_FACTOR_PAIRS : 0) | (takes_pairs(update_gemm(l)) ? ORTHO_ROUTE_UPDATE_PAIRS : 0);
}

extern "C" int aeris_orthogonalise(const AerisOrtho* p, void* stream_) {
  const AerisOrtho& a = *p;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  Layout l;
  if (const int rc = l.fill(a)) return rc;
  const bool step = a.grad != nullptr;
  if (step ? !a.momentum || !a.master : !a.x || !a.out) return -6;
  if (!(a.eps >= 1e-30) || !a.status || (l.bytes && (!a.work || !on_grid(a.work, 1024) || a.work_bytes < l.bytes))) return -7;
  char* work = reinterpret_cast<char*>(a.work);
  OrthoGroups in{}, out{};
  in.n = out.n = a.groups;
  in.numel = out.numel = a.numel;
  in.status = out.status = a.status;
  in.aligned = on_grid(step ? a.grad : a.x, !step && a.bf16 ? 8 : 16) && on_grid(a.momentum, 16);
  out.aligned = on_grid(a.out, 8) && on_grid(a.master, 16) && on_grid(a.ema, 16) && on_grid(a.weights, 8);
  long long first = 0, pack_blocks[NS_GROUPS], square_blocks[NS_GROUPS];
  for (int i = 0; i < a.groups; ++i) {
    const AerisOrthoGroup& g = a.group[i];
    if (step ? !g.offsets || g.ld != g.cols : g.ld_out < g.cols) return -8;
    if (g.offsets && a.numel <= 0) return -9;
    const int c = l.group_class[i];
    const long long n = static_cast<long long>(g.rows) * g.cols, want = (n + 8191) / 8192;
    OrthoGroup& o = in.g[i];
    o.offsets = reinterpret_cast<const long long*>(g.offsets);
    o.stride = g.stride;
    o.x_stride = l.x_stride(c);
    o.x = reinterpret_cast<__half*>(work + l.x_at[c]) + l.group_first[i] * o.x_stride;
    // one round of blocks over all matrices (four fit an SM), or so many rounds that the last one does not count
    const long long share = 4ll * num_sms() / l.count, most = share < 128 ? 128 : share < NS_PARTS ? share : NS_PARTS;
    o.parts = static_cast<int>(want < most ? want : most);
    o.partial = reinterpret_cast<double*>(work) + first * NS_PARTS;
    first += g.count;
    o.rows = g.rows;
    o.cols = g.cols;
    o.ld = g.ld;
    o.ldx = pitch(l.K[c]);
    o.behind = g.behind;
    o.count = g.count;
    o.rate = g.rate;
    square_blocks[i] = o.parts;
    pack_blocks[i] = static_cast<long long>((g.rows + 63) / 64) * ((g.cols + 63) / 64);
    if (pack_blocks[i] * g.count > 0x3fffffff) return -5;
    out.g[i] = o;
    out.g[i].blocks = static_cast<int>(pack_blocks[i]);
    if (!step) out.g[i].stride = g.out_stride, out.g[i].ld = g.ld_out;
    if (l.bytes && (l.few || (l.steps.n & 1))) out.g[i].x += l.members[c] * o.x_stride;
  }
  auto blocks = [&](const OrthoGroups& g) {
    long long n = 0;
    for (int i = 0; i < g.n; ++i) n += static_cast<long long>(g.g[i].count) * g.g[i].blocks;
    return static_cast<unsigned>(n);
  };
  const OrthoInput input = {a.x, a.bf16, a.grad, a.momentum, a.norm_sq, a.beta, a.grad_scale, a.max_norm, a.nesterov, a.zero_grad};
  const OrthoOutput output = {reinterpret_cast<__nv_bfloat16*>(a.out), a.master, a.ema, reinterpret_cast<__nv_bfloat16*>(a.weights),
                              a.decay, a.ema_beta};
  if (small(l)) {
    auto kern = step ? ortho_small_kernel<true> : ortho_small_kernel<false>;
    static std::atomic<uint64_t> done[2];
    if (!allow_smem(kern, OS_SMEM, done[step])) return -20;
    for (int i = 0; i < a.groups; ++i) in.g[i].blocks = 1;
    const int rc = launch_chained(kern, blocks(in), os_threads(l.d), OS_SMEM, stream,
                                  in, input, out, output, a.eps, a.steps);
    return rc ? rc : 1;
  }
  Products run(l, work, a.status, stream);
  if (run.rc) return run.rc;
  for (int i = 0; i < a.groups; ++i) in.g[i].blocks = static_cast<int>(square_blocks[i]);
  int rc = launch_chained(step ? ortho_squares_kernel<true> : ortho_squares_kernel<false>, blocks(in), 256, 0, stream, in, input);
  if (rc) return rc;
  for (int i = 0; i < a.groups; ++i) in.g[i].blocks = static_cast<int>(pack_blocks[i]);
  rc = launch_chained(step ? ortho_pack_kernel<true> : ortho_pack_kernel<false>, blocks(in), 256, 0, stream, in, input, a.eps);
  if (rc) return rc;
  if (l.few)
    run.few(splits_of(l, 0), a.steps);
  else
    for (int k = 0; k < l.steps.n; ++k) run.group(k & 1, l.steps.size[k]);
  if (run.rc) return run.rc;
  rc = launch_chained(step ? ortho_finish_kernel<true> : ortho_finish_kernel<false>, blocks(out), 256, 0, stream, out, output);
  return rc ? rc : run.launches + 3;
}
