// Orthogonalisation of a batch of matrices by Newton-Schulz steps, and the optimizer step that uses it.
//
//   X0 = U / max(|U|_F, eps);  S = X X^T;  X <- (a I + b S + c S^2) X, a few times, on the side with fewer rows
//
// Each step applies p(x) = a x + b x^3 + c x^5 to the singular values, which (a, b, c) below push from (0, 1] to around 1.
// All products run on the tensor cores with fp16 operands and fp32 sums. fp16 and not bf16: every factor is bounded (|X| <=
// 1.21, |S| <= 1.46, |a I + b S + c S^2| <= a), so a constant scale of 512 keeps all of them inside fp16's range, and eight
// times finer rounding matters: a rounding of the first steps is amplified like the small singular values, by up to a^5 = 485.
// Error of the result (2-norm) against 64 bits on 768 x 2048 gradients with as much, a tenth and no white noise on a spectrum
// falling like 1 / i: 1.0e-3, 2.5e-3, 4.9e-3; with bf16 operands 9.3e-3, 2.0e-2, 3.9e-2.
//
// A batch holds matrices whose shorter side is d and whose longer side is K; upright ones are transposed on the way in and
// out, so that the products see one layout: X [d, K] and symmetric factors [d, d], rows of whole 128 bytes.
#include "api.h"
#include "cluster.cuh"
#include "common.cuh"
#include "host.h"

#include <cuda_fp16.h>

namespace aeris {

constexpr float NS_A = 3.4445f, NS_B = -4.7750f, NS_C = 2.0315f;
constexpr float NS_SCALE = 512.f;             // stored = NS_SCALE * value, for X and for the [d, d] factors

constexpr int NS_PARTS = 128;                 // blocks per matrix that its squares are summed in, at most

// ------------------------------------------------------------------------------------------------ in and out
// Where matrix i of a batch lies: element offset offsets[i] (checked against [0, numel) and for ascending order) or i * stride;
// rows of pitch ld.
struct MatrixAt {
  const long long* offsets;
  long long stride, numel;
  int rows, cols, ld, behind;                 // behind: offsets[-1] is the matrix before the first one
  int aligned;                                // four elements from the buffers' starts on are one vector
  int* status;
  __device__ bool vectors(long long at) const { return aligned && cols % 4 == 0 && ld % 4 == 0 && at % 4 == 0; }
  __device__ bool find(int i, long long& at) const {
    if (!offsets) {
      at = i * stride;
      return true;
    }
    at = offsets[i];
    const long long size = static_cast<long long>(rows) * cols;
    if (at >= 0 && at + size <= numel && ((i == 0 && !behind) || at >= offsets[i - 1] + size)) return true;
    if (threadIdx.x == 0) atomicCAS(status, 0, ERR_BOUNDS);
    return false;
  }
};

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

// Sums of squares of one matrix, NS_PARTS at most, in 64 bits (squares of any fp32 values add up without overflow). An
// optimizer's momentum is brought up to date on the way: M = beta M + (1 - beta) g; what is summed is M, or beta M + (1 -
// beta) g with nesterov.
template <bool STEP>
__global__ void __launch_bounds__(256) ortho_squares_kernel(const MatrixAt m, const OrthoInput in, double* __restrict__ partial) {
  chain_point();
  long long at;
  double sum = 0;
  if (m.find(blockIdx.y, at)) {
    const float gs = STEP ? step_scale(in) : 0.f;
    auto value = [&](float g, float& mom) {
      g = clean(g * gs);
      mom = in.beta * mom + (1.f - in.beta) * g;
      return in.nesterov ? in.beta * mom + (1.f - in.beta) * g : mom;
    };
    const bool flat = m.ld == m.cols;
    const long long n = static_cast<long long>(m.rows) * m.cols;
    const long long step = static_cast<long long>(gridDim.x) * 256, first = blockIdx.x * 256ll + threadIdx.x;
    const bool four = m.vectors(at);
    if (four) {
      const int per_row = m.cols / 4;
      for (long long v = first; v < n / 4; v += step) {
        const long long e = flat ? at + 4 * v : at + v / per_row * m.ld + 4 * (v % per_row);
        float4 u;
        if (STEP) {
          const float4 g = *reinterpret_cast<const float4*>(in.grad + e);
          float4 mo = *reinterpret_cast<const float4*>(in.momentum + e);
          u = make_float4(value(g.x, mo.x), value(g.y, mo.y), value(g.z, mo.z), value(g.w, mo.w));
          *reinterpret_cast<float4*>(in.momentum + e) = mo;
        } else {
          u = in_value4(in, e);
        }
        sum += static_cast<double>(u.x) * u.x + static_cast<double>(u.y) * u.y;
        sum += static_cast<double>(u.z) * u.z + static_cast<double>(u.w) * u.w;
      }
    } else {
      for (long long v = first; v < n; v += step) {
        const long long e = flat ? at + v : at + v / m.cols * m.ld + v % m.cols;
        float u;
        if (STEP) {
          float mo = in.momentum[e];
          u = value(in.grad[e], mo);
          in.momentum[e] = mo;
        } else {
          u = in_value(in, e);
        }
        sum += static_cast<double>(u) * u;
      }
    }
  }
  __shared__ double red[8];
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 8; ++i) sum += red[i];
    partial[blockIdx.y * static_cast<long long>(gridDim.x) + blockIdx.x] = sum;
  }
}

// Normed, scaled and rounded to fp16 into X [d, K] (pitch ldx), through shared memory where the matrix is upright: one 64 x 64
// tile per block. An optimizer's value is computed again from gradient and momentum, which were read a moment before.
template <bool STEP, bool UPRIGHT>
__global__ void __launch_bounds__(256) ortho_pack_kernel(const MatrixAt m, const OrthoInput in, const double* __restrict__ partial,
                                                         int parts, double eps, __half* __restrict__ X, long long x_stride,
                                                         int ldx) {
  __shared__ float tile[UPRIGHT ? 64 : 1][65];
  __shared__ float s_scale;
  chain_point();
  long long at;
  if (!m.find(blockIdx.y, at)) return;
  if (threadIdx.x < 32) {
    double sum = 0;
    for (int i = threadIdx.x; i < parts; i += 32) sum += partial[blockIdx.y * static_cast<long long>(parts) + i];
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const double norm = sqrt(sum);
    if (threadIdx.x == 0) s_scale = static_cast<float>(NS_SCALE / (norm > eps || norm != norm ? norm : eps));
  }
  __syncthreads();
  const float scale = s_scale, gs = STEP ? step_scale(in) : 0.f;
  const int tiles_c = (m.cols + 63) / 64;
  const int r0 = blockIdx.x / tiles_c * 64, c0 = blockIdx.x % tiles_c * 64;
  const int tr = threadIdx.x >> 4, tc = (threadIdx.x & 15) * 4;
  X += blockIdx.y * x_stride;
  const bool four = m.vectors(at);
  auto value = [&](float g, float mom) {
    g = clean(g * gs);
    return scale * (in.nesterov ? in.beta * mom + (1.f - in.beta) * g : mom);
  };
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int r = r0 + tr + 16 * k, c = c0 + tc;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (r < m.rows && c < m.cols) {
      const long long e = at + static_cast<long long>(r) * m.ld + c;
      if (four) {
        if (STEP) {
          const float4 g = *reinterpret_cast<const float4*>(in.grad + e);
          const float4 mo = *reinterpret_cast<const float4*>(in.momentum + e);
          v[0] = value(g.x, mo.x); v[1] = value(g.y, mo.y); v[2] = value(g.z, mo.z); v[3] = value(g.w, mo.w);
          if (in.zero_grad) *reinterpret_cast<float4*>(in.grad + e) = make_float4(0.f, 0.f, 0.f, 0.f);
        } else {
          const float4 u = in_value4(in, e);
          v[0] = scale * u.x; v[1] = scale * u.y; v[2] = scale * u.z; v[3] = scale * u.w;
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (c + j >= m.cols) break;
          if (STEP) {
            v[j] = value(in.grad[e + j], in.momentum[e + j]);
            if (in.zero_grad) in.grad[e + j] = 0.f;
          } else {
            v[j] = scale * in_value(in, e + j);
          }
        }
      }
    }
    if (UPRIGHT) {
#pragma unroll
      for (int j = 0; j < 4; ++j) tile[tr + 16 * k][tc + j] = v[j];
    } else if (r < m.rows && c < ldx) {
      __half2 h[2] = {__floats2half2_rn(v[0], v[1]), __floats2half2_rn(v[2], v[3])};
      *reinterpret_cast<uint2*>(X + static_cast<long long>(r) * ldx + c) = *reinterpret_cast<uint2*>(h);
    }
  }
  if (UPRIGHT) {
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int r = c0 + tr + 16 * k, c = r0 + tc;          // row and column of X
      if (r < m.cols && c < ldx) {
        __half2 h[2] = {__floats2half2_rn(tile[tc][tr + 16 * k], tile[tc + 1][tr + 16 * k]),
                        __floats2half2_rn(tile[tc + 2][tr + 16 * k], tile[tc + 3][tr + 16 * k])};
        *reinterpret_cast<uint2*>(X + static_cast<long long>(r) * ldx + c) = *reinterpret_cast<uint2*>(h);
      }
    }
  }
}

// What becomes of the orthogonalised matrices: a bf16 tensor, or the update of an optimizer's weights.
struct OrthoOutput {
  __nv_bfloat16* out;
  float *master, *ema;                        // optimizer: master set
  __nv_bfloat16* weights;                     // may be null
  float decay, rate, ema_beta;                // master * decay - rate * X; ema_beta < 0: no running average
};

template <bool STEP, bool UPRIGHT>
__global__ void __launch_bounds__(256) ortho_finish_kernel(const MatrixAt m, const OrthoOutput o, const __half* __restrict__ X,
                                                           long long x_stride, int ldx, const int* status) {
  __shared__ float tile[UPRIGHT ? 64 : 1][65];
  chain_point();
  long long at;
  if (!m.find(blockIdx.y, at) || failed(status)) return;      // what a kernel that gave up left behind is not applied
  const int tiles_c = (m.cols + 63) / 64;
  const int r0 = blockIdx.x / tiles_c * 64, c0 = blockIdx.x % tiles_c * 64;
  const int tr = threadIdx.x >> 4, tc = (threadIdx.x & 15) * 4;
  X += blockIdx.y * x_stride;
  if (UPRIGHT) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int r = c0 + tr + 16 * k, c = r0 + tc;
      if (r < m.cols && c < ldx) {
        const uint2 w = *reinterpret_cast<const uint2*>(X + static_cast<long long>(r) * ldx + c);
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x));
        const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
        tile[tc][tr + 16 * k] = a.x; tile[tc + 1][tr + 16 * k] = a.y;
        tile[tc + 2][tr + 16 * k] = b.x; tile[tc + 3][tr + 16 * k] = b.y;
      }
    }
    __syncthreads();
  }
  const bool four = m.vectors(at);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int r = r0 + tr + 16 * k, c = c0 + tc;
    if (r >= m.rows || c >= m.cols) continue;
    const long long e = at + static_cast<long long>(r) * m.ld + c;
    float v[4];
    if (UPRIGHT) {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = tile[tr + 16 * k][tc + j];
    } else {
      const uint2 w = *reinterpret_cast<const uint2*>(X + static_cast<long long>(r) * ldx + c);
      const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x));
      const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
      v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] *= 1.f / NS_SCALE;
    if (!STEP) {
      if (four) {
        *reinterpret_cast<uint2*>(o.out + e) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
      } else {
        for (int j = 0; j < 4 && c + j < m.cols; ++j) o.out[e + j] = __float2bfloat16_rn(v[j]);
      }
      continue;
    }
    if (four) {
      const float4 p4 = *reinterpret_cast<const float4*>(o.master + e);
      const float p[4] = {p4.x * o.decay - o.rate * v[0], p4.y * o.decay - o.rate * v[1], p4.z * o.decay - o.rate * v[2],
                          p4.w * o.decay - o.rate * v[3]};
      *reinterpret_cast<float4*>(o.master + e) = make_float4(p[0], p[1], p[2], p[3]);
      if (o.weights) *reinterpret_cast<uint2*>(o.weights + e) = make_uint2(pack_bf16x2(p[0], p[1]), pack_bf16x2(p[2], p[3]));
      if (o.ema && o.ema_beta >= 0.f) {
        float4 a = *reinterpret_cast<const float4*>(o.ema + e);
        a.x = p[0] + o.ema_beta * (a.x - p[0]); a.y = p[1] + o.ema_beta * (a.y - p[1]);
        a.z = p[2] + o.ema_beta * (a.z - p[2]); a.w = p[3] + o.ema_beta * (a.w - p[3]);
        *reinterpret_cast<float4*>(o.ema + e) = a;
      }
    } else {
      for (int j = 0; j < 4 && c + j < m.cols; ++j) {
        const float p = o.master[e + j] * o.decay - o.rate * v[j];
        o.master[e + j] = p;
        if (o.weights) o.weights[e + j] = __float2bfloat16_rn(p);
        if (o.ema && o.ema_beta >= 0.f) o.ema[e + j] = p + o.ema_beta * (o.ema[e + j] - p);
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------ products
// C = alpha A B^T + beta R + gamma I for every matrix of a batch (B stored [K, N] with B_MN); fp16 in and out, fp32 sums.
// `sym`: the result is symmetric, only tiles on and below the diagonal are computed and the others are their mirror images.
// One CTA per 128 x 128 tile at a time: a TMA producer, an issuer of tcgen05.mma, four epilogue warps, two accumulators.
struct OrthoGemm {
  int M, N, K, count, sym;
  int a0, b0;                                 // first matrix of the batch in the operands' tensor maps
  __half* C;
  const __half* R;                            // null, or laid out like C
  long long c_stride;
  int ldc;
  float alpha, beta, gamma;
  int* status;
};

constexpr int OG_TILE = 128, OG_BK = 64, OG_STAGES = 6, OG_THREADS = 192;
constexpr int OG_OPERAND = OG_TILE * OG_BK * 2;
constexpr int OG_STAGE = 2 * OG_OPERAND;
constexpr int OG_SMEM = OG_STAGES * OG_STAGE + 256 + 1024;

__device__ __forceinline__ void tma_load_3d(void* smem_dst, const CUtensorMap* m, uint64_t* bar, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
          smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
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

// Tile `t` of one matrix: row by row, or the t-th on and below the diagonal.
__device__ __forceinline__ void ortho_tile(int t, int sym, int n_tiles, int& ti, int& tj) {
  if (!sym) {
    ti = t / n_tiles;
    tj = t - ti * n_tiles;
    return;
  }
  ti = static_cast<int>((sqrtf(8.f * t + 1.f) - 1.f) * 0.5f);
  while (ti * (ti + 1) / 2 > t) --ti;
  while ((ti + 1) * (ti + 2) / 2 <= t) ++ti;
  tj = t - ti * (ti + 1) / 2;
}

// One thread's row of a tile: NCOL accumulator columns from `taddr` on are columns col0 .. of row `row`.
template <int NCOL>
__device__ __forceinline__ void ortho_epilogue(const OrthoGemm& p, uint32_t taddr, int mat, int row, int col0, bool keep,
                                               bool mirror) {
  const long long at = mat * p.c_stride;
  __half* C = p.C + at;
  const __half* R = p.R ? p.R + at : nullptr;
#pragma unroll 1
  for (int c = 0; c < NCOL; c += 32) {
    const int col = col0 + c;
    if (col >= p.ldc) break;
    uint32_t v[32];
    tmem_ld32(taddr + c, v);
    tmem_wait_ld();
    if (!keep || row >= p.M) continue;
    float f[32];
#pragma unroll
    for (int j = 0; j < 32; ++j) f[j] = p.alpha * __uint_as_float(v[j]);
    if (R) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint4 w = *reinterpret_cast<const uint4*>(R + static_cast<long long>(row) * p.ldc + col + 8 * j);
        const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 r2 = __half22float2(*reinterpret_cast<const __half2*>(&ww[i]));
          f[8 * j + 2 * i] += p.beta * r2.x;
          f[8 * j + 2 * i + 1] += p.beta * r2.y;
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (row == col + j) f[j] += p.gamma;
    __half2 h[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) h[j] = __floats2half2_rn(f[2 * j], f[2 * j + 1]);
    uint4* dst = reinterpret_cast<uint4*>(C + static_cast<long long>(row) * p.ldc + col);
#pragma unroll
    for (int j = 0; j < 4; ++j) dst[j] = reinterpret_cast<uint4*>(h)[j];
    if (p.sym && mirror) {                 // the mirror image: for one column after the other, 32 rows side by side
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (col + j < p.N) C[static_cast<long long>(col + j) * p.ldc + row] = j & 1 ? __high2half(h[j / 2]) : __low2half(h[j / 2]);
    }
  }
}

template <int B_MN>
__global__ void __launch_bounds__(OG_THREADS, 1)
ortho_gemm_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b, const OrthoGemm p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + OG_STAGES * OG_STAGE);
  uint64_t* empty_bar = full_bar + OG_STAGES;
  uint64_t* tfull_bar = empty_bar + OG_STAGES;
  uint64_t* tempty_bar = tfull_bar + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty_bar + 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int m_tiles = (p.M + OG_TILE - 1) / OG_TILE, n_tiles = (p.N + OG_TILE - 1) / OG_TILE;
  const int per_matrix = p.sym ? m_tiles * (m_tiles + 1) / 2 : m_tiles * n_tiles;
  const int total = per_matrix * p.count;
  const int kb_total = (p.K + OG_BK - 1) / OG_BK;
  if (threadIdx.x == 0) {
    prefetch_tmap(&tmap_a);
    prefetch_tmap(&tmap_b);
    for (int s = 0; s < OG_STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull_bar[a], 1);
      mbar_init(&tempty_bar[a], 4);
    }
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 2 * OG_TILE);
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
      for (int tile = blockIdx.x; tile < total && ok; tile += gridDim.x) {
        const int mat = tile / per_matrix;
        int ti, tj;
        ortho_tile(tile - mat * per_matrix, p.sym, n_tiles, ti, tj);
        for (int kb = 0; kb < kb_total; ++kb) {
          if (!own_wait(&empty_bar[stage], phase ^ 1, p.status, ERR_TIMEOUT_EMPTY)) { ok = false; break; }
          uint8_t* sa = smem + stage * OG_STAGE;
          uint8_t* sb = sa + OG_OPERAND;
          mbar_expect_tx(&full_bar[stage], OG_STAGE);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            tma_load_3d(sa + j * 8192, &tmap_a, &full_bar[stage], kb * OG_BK, ti * OG_TILE + j * 64, p.a0 + mat);
            if (B_MN)
              tma_load_3d(sb + j * 8192, &tmap_b, &full_bar[stage], tj * OG_TILE + j * 64, kb * OG_BK, p.b0 + mat);
            else
              tma_load_3d(sb + j * 8192, &tmap_b, &full_bar[stage], kb * OG_BK, tj * OG_TILE + j * 64, p.b0 + mat);
          }
          if (++stage == OG_STAGES) { stage = 0; phase ^= 1; }
        }
      }
      // every stage filled has been consumed, or at least arrived, before the CTA leaves
      for (int s = 0; s < OG_STAGES; ++s) {
        if (ok) {
          if (!own_wait(&empty_bar[stage], phase ^ 1, p.status, ERR_TIMEOUT_EMPTY)) break;
          if (++stage == OG_STAGES) { stage = 0; phase ^= 1; }
        } else {
          if (--stage < 0) { stage = OG_STAGES - 1; phase ^= 1; }
          if (!own_wait(&full_bar[stage], phase, nullptr, 0)) break;
        }
      }
    }
  } else if (warp == 1) {
    if (elect_one_sync()) {
      constexpr uint32_t idesc = make_idesc_fp16(OG_TILE, OG_TILE, B_MN);
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int tile = blockIdx.x; tile < total && ok; tile += gridDim.x) {
        if (!own_wait(&tempty_bar[acc], acc_phase ^ 1, p.status, ERR_TIMEOUT_TMEM_EMPTY)) break;
        tc_fence_after();
        const uint32_t tmem_acc = tmem_base + acc * OG_TILE;
        for (int kb = 0; kb < kb_total; ++kb) {
          if (!own_wait(&full_bar[stage], phase, p.status, ERR_TIMEOUT_FULL)) { ok = false; break; }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + stage * OG_STAGE), sb = sa + OG_OPERAND;
#pragma unroll
          for (int kk = 0; kk < OG_BK / 16; ++kk)
            umma_ss(tmem_acc, make_smem_desc(sa + kk * 32, 0, 1024),
                    B_MN ? make_smem_desc(sb + kk * 2048, 8192, 1024) : make_smem_desc(sb + kk * 32, 0, 1024), idesc,
                    kb > 0 || kk > 0);
          tc_commit(&empty_bar[stage]);
          if (++stage == OG_STAGES) { stage = 0; phase ^= 1; }
        }
        if (!ok) break;
        tc_commit(&tfull_bar[acc]);
        if (++acc == 2) { acc = 0; acc_phase ^= 1; }
      }
      // the last products have completed before the tensor memory goes back (a stage never filled counts as done)
      if (--stage < 0) { stage = OG_STAGES - 1; phase ^= 1; }
      own_wait(&empty_bar[stage], phase, nullptr, 0);
    }
  } else {
    const int q = warp & 3;
    int acc = 0;
    uint32_t acc_phase = 0;
    const bool keep = !failed(p.status);
    for (int tile = blockIdx.x; tile < total; tile += gridDim.x) {
      const int mat = tile / per_matrix;
      int ti, tj;
      ortho_tile(tile - mat * per_matrix, p.sym, n_tiles, ti, tj);
      if (!__all_sync(0xffffffffu, own_wait(&tfull_bar[acc], acc_phase, p.status, ERR_TIMEOUT_TMEM_FULL))) break;
      tc_fence_after();
      const int row = ti * OG_TILE + q * 32 + lane;
      const uint32_t taddr = tmem_base + acc * OG_TILE + (static_cast<uint32_t>(q * 32) << 16);
      ortho_epilogue<OG_TILE>(p, taddr, mat, row, tj * OG_TILE, keep, ti != tj);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tempty_bar[acc]);
      if (++acc == 2) { acc = 0; acc_phase ^= 1; }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem_base, 2 * OG_TILE);
}

// The same on CTA pairs: a cluster of two computes a 256 x 256 tile, each CTA staging its 128 rows of A and half of B's columns
// (csrc/gemm2.cu has the scheme). Per product a third less shared memory and L2 traffic than a 128 x 128 tile needs half of.
constexpr int OP_BM = 128, OP_BN = 256, OP_STAGES = 6;
constexpr int OP_OPERAND = 128 * OG_BK * 2;
constexpr int OP_STAGE = 2 * OP_OPERAND;
constexpr int OP_SMEM = OP_STAGES * OP_STAGE + 256 + 1024;

template <int B_MN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(OG_THREADS, 1)
ortho_gemm_pair_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b, const OrthoGemm p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + OP_STAGES * OP_STAGE);      // the leader's: both CTAs' bytes
  uint64_t* empty_bar = full_bar + OP_STAGES;
  uint64_t* tfull_bar = empty_bar + OP_STAGES;
  uint64_t* tempty_bar = tfull_bar + 2;                                               // the leader's: both CTAs' warps
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty_bar + 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t crank = cluster_ctarank();
  const int cluster = blockIdx.x >> 1, clusters = gridDim.x >> 1;
  const int m_tiles = (p.M + 2 * OP_BM - 1) / (2 * OP_BM), n_tiles = (p.N + OP_BN - 1) / OP_BN;
  const int per_matrix = p.sym ? m_tiles * (m_tiles + 1) / 2 : m_tiles * n_tiles;
  const int total = per_matrix * p.count;
  const int kb_total = (p.K + OG_BK - 1) / OG_BK;
  if (threadIdx.x == 0) {
    prefetch_tmap(&tmap_a);
    prefetch_tmap(&tmap_b);
    for (int s = 0; s < OP_STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull_bar[a], 1);
      mbar_init(&tempty_bar[a], 8);
    }
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc2(tmem_slot, 2 * OP_BN);
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
      for (int tile = cluster; tile < total && ok; tile += clusters) {
        const int mat = tile / per_matrix;
        int ti, tj;
        ortho_tile(tile - mat * per_matrix, p.sym, n_tiles, ti, tj);
        const int m0 = ti * 2 * OP_BM + crank * OP_BM, n0 = tj * OP_BN + crank * (OP_BN / 2);
        for (int kb = 0; kb < kb_total; ++kb) {
          if (!own_poll(&empty_bar[stage], phase ^ 1, p.status, ERR_TIMEOUT_EMPTY)) { ok = false; break; }
          uint8_t* sa = smem + stage * OP_STAGE;
          uint8_t* sb = sa + OP_OPERAND;
          if (crank == 0) mbar_expect_tx(&full_bar[stage], 2 * OP_STAGE);
          const uint32_t fb = map_to_cta(smem_u32(&full_bar[stage]), 0);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            tma_load_3d_pair(sa + j * 8192, &tmap_a, fb, kb * OG_BK, m0 + j * 64, p.a0 + mat);
            if (B_MN)
              tma_load_3d_pair(sb + j * 8192, &tmap_b, fb, n0 + j * 64, kb * OG_BK, p.b0 + mat);
            else
              tma_load_3d_pair(sb + j * 8192, &tmap_b, fb, kb * OG_BK, n0 + j * 64, p.b0 + mat);
          }
          if (++stage == OP_STAGES) { stage = 0; phase ^= 1; }
        }
      }
      // tiles that the issuer did not take, of both CTAs (a stage never filled counts as there)
      for (int s = 0; s < OP_STAGES && !ok && crank == 0; ++s) {
        if (--stage < 0) { stage = OP_STAGES - 1; phase ^= 1; }
        if (!own_poll(&full_bar[stage], phase, nullptr, 0)) break;
      }
    }
  } else if (warp == 1) {
    if (crank == 0 && elect_one_sync()) {
      constexpr uint32_t idesc = make_idesc_fp16(2 * OP_BM, OP_BN, B_MN);
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int tile = cluster; tile < total && ok; tile += clusters) {
        if (!own_poll(&tempty_bar[acc], acc_phase ^ 1, p.status, ERR_TIMEOUT_TMEM_EMPTY)) break;
        tc_fence_after();
        const uint32_t tmem_acc = tmem_base + acc * OP_BN;
        for (int kb = 0; kb < kb_total; ++kb) {
          if (!own_poll(&full_bar[stage], phase, p.status, ERR_TIMEOUT_FULL)) { ok = false; break; }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + stage * OP_STAGE), sb = sa + OP_OPERAND;
#pragma unroll
          for (int kk = 0; kk < OG_BK / 16; ++kk)
            umma2_ss(tmem_acc, make_smem_desc(sa + kk * 32, 0, 1024),
                     B_MN ? make_smem_desc(sb + kk * 2048, 8192, 1024) : make_smem_desc(sb + kk * 32, 0, 1024), idesc,
                     kb > 0 || kk > 0);
          tc_commit2_mc(&empty_bar[stage], 0x3);
          if (++stage == OP_STAGES) { stage = 0; phase ^= 1; }
        }
        if (!ok) break;
        tc_commit2_mc(&tfull_bar[acc], 0x3);
        if (++acc == 2) { acc = 0; acc_phase ^= 1; }
      }
      // the last products have completed before the CTAs leave
      if (--stage < 0) { stage = OP_STAGES - 1; phase ^= 1; }
      own_poll(&empty_bar[stage], phase, nullptr, 0);
    }
  } else {
    const int q = warp & 3;
    int acc = 0;
    uint32_t acc_phase = 0;
    const bool keep = !failed(p.status);
    const uint32_t leader_tempty = map_to_cta(smem_u32(&tempty_bar[0]), 0);
    for (int tile = cluster; tile < total; tile += clusters) {
      const int mat = tile / per_matrix;
      int ti, tj;
      ortho_tile(tile - mat * per_matrix, p.sym, n_tiles, ti, tj);
      if (!__all_sync(0xffffffffu, own_poll(&tfull_bar[acc], acc_phase, p.status, ERR_TIMEOUT_TMEM_FULL))) break;
      tc_fence_after();
      const int row = ti * 2 * OP_BM + crank * OP_BM + q * 32 + lane;
      ortho_epilogue<OP_BN>(p, tmem_base + acc * OP_BN + (static_cast<uint32_t>(q * 32) << 16), mat, row, tj * OP_BN, keep,
                            ti != tj);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_remote(leader_tempty + acc * 8);
      if (++acc == 2) { acc = 0; acc_phase ^= 1; }
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  tc_fence_after();
  if (warp == 1) tmem_dealloc2(tmem_base, 2 * OP_BN);
}

// ------------------------------------------------------------------------------------------------ host side
namespace {

int pitch(int n) { return (n + 63) / 64 * 64; }
bool on_grid(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// How the steps are grouped. One step by itself is a Gram matrix of X, its square and an update of X: in units of d^3, with
// symmetric products at half and r = K / d, 3 r + 1. Two steps can share the update: the Gram matrix alone goes on (S <- P S P
// with P = a I + b S + c S^2, all symmetric and commuting) and X is multiplied by the product of both P at the end: 3 r + 5
// instead of 6 r + 2, the less for every oblong matrix. Groups of three would cost 3 r + 9, but a Gram matrix's rounding error
// (2^-12 of its norm) grows by a^2 a step in directions that hold little of the norm, and is not small against them any more:
// error on 127 x 640 gradients with half as much noise as signal 6e-4 by single steps and in groups (2, 2, 1), 1.8e-3 in (3, 2); on
// 320 x 2000 5.5e-4, 6.5e-4, 9e-4; a group of five diverges. Below GROUP_FROM rows single steps: the products are shorter than
// their launches, of which groups have two more, and a handful of rows does not average the roundings (5 x 9: up to three times
// the error of single steps).
constexpr int GROUP_FROM = 256;
struct Groups {
  int n, size[20];
};
Groups groups_of(int d, int K, int steps) {
  Groups g = {0, {}};
  for (int left = steps, most = K > d && d >= GROUP_FROM ? 2 : 1; left > 0; left -= g.size[g.n++]) g.size[g.n] = left < most ? left : most;
  return g;
}
int buffers_of(const Groups& g) { return g.size[0] == 1 ? 2 : 4; }

enum Factor { F_S, F_P0, F_T, F_P1 };    // where the [d, d] factors of a batch are

struct Products {
  CUtensorMap x, s;                           // 2 * count matrices X, and all factors
  __half *X, *S;
  int count, d, K;
  int* status;
  cudaStream_t stream;
  int launches = 0, rc = 0;

  long long x_stride() const { return static_cast<long long>(d) * pitch(K); }
  long long s_stride() const { return static_cast<long long>(d) * pitch(d); }
  __half* at(int f) const { return S + f * count * s_stride(); }

  template <int B_MN>
  void launch(const CUtensorMap& a, const CUtensorMap& b, OrthoGemm p) {
    if (rc) return;
    static bool configured = false;
    if (!configured) {
      if (cudaFuncSetAttribute(ortho_gemm_kernel<B_MN>, cudaFuncAttributeMaxDynamicSharedMemorySize, OG_SMEM) != cudaSuccess ||
          cudaFuncSetAttribute(ortho_gemm_pair_kernel<B_MN>, cudaFuncAttributeMaxDynamicSharedMemorySize, OP_SMEM) != cudaSuccess) {
        rc = -20;
        return;
      }
      configured = true;
    }
    p.count = count;
    p.status = status;
    auto tiles_of = [&](int tile) {
      const long long m = (p.M + tile - 1) / tile, n = (p.N + tile - 1) / tile;
      return (p.sym ? m * (m + 1) / 2 : m * n) * count;
    };
    const long long small = tiles_of(OG_TILE), large = tiles_of(2 * OG_TILE);
    if (small > 0x7fffffff) {
      rc = -5;
      return;
    }
    // rounds of tiles; a pair's tile has twice the work per multiprocessor of a single one's and takes about as long
    const int sms = num_sms(), pairs = sms / 2;
    if ((large + pairs - 1) / pairs <= (small + sms - 1) / sms)
      rc = launch_chained(ortho_gemm_pair_kernel<B_MN>, 2 * static_cast<int>(large < pairs ? large : pairs), OG_THREADS, OP_SMEM,
                          stream, a, b, p);
    else
      rc = launch_chained(ortho_gemm_kernel<B_MN>, static_cast<int>(small < sms ? small : sms), OG_THREADS, OG_SMEM, stream, a, b,
                          p);
    ++launches;
  }
  void product(int out, int i, int j) {       // factor `out` = (factor i) (factor j)
    OrthoGemm p{};
    p.M = p.N = p.K = d;
    p.sym = 1;
    p.a0 = i * count;
    p.b0 = j * count;
    p.C = at(out);
    p.c_stride = s_stride();
    p.ldc = pitch(d);
    p.alpha = 1.f / NS_SCALE;
    launch<0>(s, s, p);
  }
  void polynomial(int out) {                  // factor `out` = a I + b S + c S^2
    OrthoGemm p{};
    p.M = p.N = p.K = d;
    p.sym = 1;
    p.a0 = p.b0 = F_S * count;
    p.C = at(out);
    p.R = at(F_S);
    p.c_stride = s_stride();
    p.ldc = pitch(d);
    p.alpha = NS_C / NS_SCALE;
    p.beta = NS_B;
    p.gamma = NS_A * NS_SCALE;
    launch<0>(s, s, p);
  }
  void gram(int from) {                       // S = X X^T
    OrthoGemm p{};
    p.M = p.N = d;
    p.K = K;
    p.sym = 1;
    p.a0 = p.b0 = from * count;
    p.C = at(F_S);
    p.c_stride = s_stride();
    p.ldc = pitch(d);
    p.alpha = 1.f / NS_SCALE;
    launch<0>(x, x, p);
  }
  void update(int from, int by) {             // the other X = factor `by` X
    OrthoGemm p{};
    p.M = p.K = d;
    p.N = K;
    p.a0 = by * count;
    p.b0 = from * count;
    p.C = X + (1 - from) * count * x_stride();
    p.c_stride = x_stride();
    p.ldc = pitch(K);
    p.alpha = 1.f / NS_SCALE;
    launch<1>(s, x, p);
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

extern "C" int aeris_ortho_buffers(int d, int K, int steps) {
  return d <= 0 || K < d || steps < 1 || steps > 20 ? -1 : buffers_of(groups_of(d, K, steps));
}

extern "C" int aeris_ortho_updates(int d, int K, int steps) {
  return d <= 0 || K < d || steps < 1 || steps > 20 ? -1 : groups_of(d, K, steps).n;
}

extern "C" int aeris_ortho_in(const AerisOrthoIn* a, void* stream_) {
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  const bool step = a->grad != nullptr;
  if (a->count <= 0 || a->count > 65535 || a->rows <= 0 || a->cols <= 0 || a->ld < a->cols || !a->X || !a->partial) return -1;
  if (step ? !a->momentum || !a->offsets || a->ld != a->cols : !a->x) return -2;
  if (a->offsets && (!a->status || a->numel <= 0)) return -3;
  const long long n = static_cast<long long>(a->rows) * a->cols;
  const long long want = (n + 4095) / 4096;
  const int parts = static_cast<int>(want < NS_PARTS ? want : NS_PARTS);
  const long long tiles = static_cast<long long>((a->rows + 63) / 64) * ((a->cols + 63) / 64);
  if (tiles > 0x7fffffff) return -5;
  const int aligned = on_grid(step ? a->grad : a->x, !step && a->bf16 ? 8 : 16) && on_grid(a->momentum, 16);
  const MatrixAt m = {reinterpret_cast<const long long*>(a->offsets), a->stride, a->numel, a->rows, a->cols, a->ld, a->behind,
                      aligned, a->status};
  const OrthoInput in = {a->x, a->bf16, a->grad, a->momentum, a->norm_sq, a->beta, a->grad_scale, a->max_norm, a->nesterov,
                         a->zero_grad};
  const bool upright = a->rows > a->cols;
  const int d = upright ? a->cols : a->rows, ldx = pitch(upright ? a->rows : a->cols);
  const long long x_stride = static_cast<long long>(d) * ldx;
  __half* X = reinterpret_cast<__half*>(a->X);
  const int rc = launch_chained(step ? ortho_squares_kernel<true> : ortho_squares_kernel<false>, dim3(parts, a->count), 256, 0,
                                stream, m, in, a->partial);
  if (rc) return rc;
  auto pack = step ? (upright ? ortho_pack_kernel<true, true> : ortho_pack_kernel<true, false>)
                   : (upright ? ortho_pack_kernel<false, true> : ortho_pack_kernel<false, false>);
  return launch_chained(pack, dim3(static_cast<unsigned>(tiles), a->count), 256, 0, stream, m, in,
                        static_cast<const double*>(a->partial), parts, a->eps, X, x_stride, ldx);
}

extern "C" int aeris_ortho_iterate(void* X, void* S, int count, int d, int K, int steps, int* status, void* stream) {
  if (!X || !S || !status || count <= 0 || d <= 0 || K < d || steps < 1 || steps > 20) return -1;
  const Groups groups = groups_of(d, K, steps);
  Products p;
  p.X = reinterpret_cast<__half*>(X);
  p.S = reinterpret_cast<__half*>(S);
  p.count = count;
  p.d = d;
  p.K = K;
  p.status = status;
  p.stream = reinterpret_cast<cudaStream_t>(stream);
  if (const int r = make_tmap_3d_fp16(&p.x, X, K, d, 2ull * count, pitch(K), 64)) return r;
  if (const int r = make_tmap_3d_fp16(&p.s, S, d, d, static_cast<uint64_t>(buffers_of(groups)) * count, pitch(d), 64)) return r;
  for (int k = 0; k < groups.n; ++k) p.group(k & 1, groups.size[k]);
  return p.rc ? p.rc : p.launches;
}

extern "C" int aeris_ortho_out(const AerisOrthoOut* a, void* stream_) {
  const bool step = a->master != nullptr;
  if (a->count <= 0 || a->count > 65535 || a->rows <= 0 || a->cols <= 0 || a->ld < a->cols || !a->X || !a->status) return -1;
  if (step ? !a->offsets || a->ld != a->cols : !a->out) return -2;
  if (a->offsets && a->numel <= 0) return -3;
  const long long tiles = static_cast<long long>((a->rows + 63) / 64) * ((a->cols + 63) / 64);
  if (tiles > 0x7fffffff) return -5;
  const int aligned = on_grid(a->out, 8) && on_grid(a->master, 16) && on_grid(a->ema, 16) && on_grid(a->weights, 8);
  const MatrixAt m = {reinterpret_cast<const long long*>(a->offsets), a->stride, a->numel, a->rows, a->cols, a->ld, a->behind,
                      aligned, a->status};
  const OrthoOutput o = {reinterpret_cast<__nv_bfloat16*>(a->out), a->master, a->ema, reinterpret_cast<__nv_bfloat16*>(a->weights),
                         a->decay, a->rate, a->ema_beta};
  const bool upright = a->rows > a->cols;
  const int d = upright ? a->cols : a->rows, ldx = pitch(upright ? a->rows : a->cols);
  auto kern = step ? (upright ? ortho_finish_kernel<true, true> : ortho_finish_kernel<true, false>)
                   : (upright ? ortho_finish_kernel<false, true> : ortho_finish_kernel<false, false>);
  return launch_chained(kern, dim3(static_cast<unsigned>(tiles), a->count), 256, 0, reinterpret_cast<cudaStream_t>(stream_), m, o,
                        reinterpret_cast<const __half*>(a->X), static_cast<long long>(d) * ldx, ldx,
                        static_cast<const int*>(a->status));
}
