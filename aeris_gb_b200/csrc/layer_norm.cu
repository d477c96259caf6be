// Layer norm over the columns of a row, forward and backward.
//
//   mean = sum x / n, var = sum (x - mean)^2 / n, rstd = 1 / sqrt(var + eps), xhat = (x - mean) rstd
//   y = xhat w + b
//   g = dy w, dx = rstd (g - mean(g) - xhat mean(g xhat)), dw = sum dy xhat, db = sum dy         (sums over rows)
//
// Statistics and sums are fp32 whatever the tensors' type; the variance is taken around the mean (two passes over the row), not
// as a difference of two large sums. Results are rounded once.
#include "common.cuh"
#include "api.h"
#include "host.h"
#include "cluster.cuh"

namespace aeris {

namespace {

constexpr int LN_THREADS = 256;
constexpr int LN_COLS = 64;        // columns of a block of the column sums

__device__ __forceinline__ float ld_f(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float ld_f(const float* p) { return *p; }
__device__ __forceinline__ void st_f(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void st_f(float* p, float v) { *p = v; }

__device__ __forceinline__ float weight_at(const void* w, int f32, int c) {
  return f32 ? static_cast<const float*>(w)[c] : __bfloat162float(static_cast<const __nv_bfloat16*>(w)[c]);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Sum over the block, in every thread; `part` [32] may be used again after the next call's first barrier.
__device__ __forceinline__ float block_sum(float v, float* part) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = (threadIdx.x & 31) < blockDim.x / 32 ? part[threadIdx.x & 31] : 0.f;
  return warp_sum(v);
}

// Any width (what layer_norm_fast.cuh does not hold in registers): a block per row, which it reads three times.
template <typename T>
__global__ void __launch_bounds__(LN_THREADS) ln_fwd_any_kernel(const AerisLayerNorm a) {
  __shared__ float part[32];
  chain_point();
  const long long row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.ld_x;
  T* y = static_cast<T*>(a.y) + row * a.ld_y;
  const float inv = 1.f / static_cast<float>(a.cols);
  float s = 0.f;
  for (int c = threadIdx.x; c < a.cols; c += LN_THREADS) s += ld_f(x + c);
  const float mean = block_sum(s, part) * inv;
  s = 0.f;
  for (int c = threadIdx.x; c < a.cols; c += LN_THREADS) {
    const float d = ld_f(x + c) - mean;
    s = fmaf(d, d, s);
  }
  const float rstd = 1.f / sqrtf(block_sum(s, part) * inv + a.eps);
  for (int c = threadIdx.x; c < a.cols; c += LN_THREADS) {
    float v = (ld_f(x + c) - mean) * rstd;
    if (a.w) v *= weight_at(a.w, a.w_f32, c);
    if (a.b) v += weight_at(a.b, a.w_f32, c);
    st_f(y + c, v);
  }
  if (threadIdx.x == 0) {
    a.stats[2 * row] = mean;
    a.stats[2 * row + 1] = rstd;
  }
}

template <typename T>
__global__ void __launch_bounds__(LN_THREADS) ln_bwd_any_kernel(const AerisLayerNorm a) {
  __shared__ float part[32];
  chain_point();
  const long long row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.ld_x;
  const T* dy = static_cast<const T*>(a.dy) + row * a.ld_dy;
  T* dx = static_cast<T*>(a.y) + row * a.ld_y;
  const float mean = a.stats[2 * row], rstd = a.stats[2 * row + 1], inv = 1.f / static_cast<float>(a.cols);
  float s1 = 0.f, s2 = 0.f;
  for (int c = threadIdx.x; c < a.cols; c += LN_THREADS) {
    const float g = ld_f(dy + c) * (a.w ? weight_at(a.w, a.w_f32, c) : 1.f);
    s1 += g;
    s2 = fmaf(g, (ld_f(x + c) - mean) * rstd, s2);
  }
  s1 = block_sum(s1, part) * inv;
  s2 = block_sum(s2, part) * inv;
  for (int c = threadIdx.x; c < a.cols; c += LN_THREADS) {
    const float g = ld_f(dy + c) * (a.w ? weight_at(a.w, a.w_f32, c) : 1.f);
    st_f(dx + c, rstd * (g - s1 - (ld_f(x + c) - mean) * rstd * s2));
  }
}

// Column sums of one slice of the rows: blocks of 64 columns by 4 rows at a time, joined in shared memory.
template <typename T>
__global__ void __launch_bounds__(LN_THREADS) ln_sums_any_kernel(const AerisLayerNorm a) {
  __shared__ float part[2][LN_THREADS];
  chain_point();
  constexpr int R = LN_THREADS / LN_COLS;
  const int c = blockIdx.x * LN_COLS + threadIdx.x % LN_COLS, r0 = threadIdx.x / LN_COLS;
  float dw = 0.f, db = 0.f;
  if (c < a.cols)
    for (long long row = static_cast<long long>(blockIdx.y) * R + r0; row < a.rows; row += static_cast<long long>(a.slices) * R) {
      const float dy = ld_f(static_cast<const T*>(a.dy) + row * a.ld_dy + c);
      const float x = ld_f(static_cast<const T*>(a.x) + row * a.ld_x + c);
      dw = fmaf(dy, (x - a.stats[2 * row]) * a.stats[2 * row + 1], dw);
      db += dy;
    }
  part[0][threadIdx.x] = dw;
  part[1][threadIdx.x] = db;
  __syncthreads();
  if (threadIdx.x < 2 * LN_COLS) {
    const int which = threadIdx.x / LN_COLS, k = threadIdx.x % LN_COLS, col = blockIdx.x * LN_COLS + k;
    float s = 0.f;
#pragma unroll
    for (int r = 0; r < R; ++r) s += part[which][r * LN_COLS + k];
    if (col < a.cols) a.work[(static_cast<long long>(blockIdx.y) * 2 + which) * a.cols + col] = s;
  }
}

// dw, db from the slices' sums: 32 columns by 32 warps, which share the slices.
__global__ void __launch_bounds__(1024) ln_join_kernel(const AerisLayerNorm a, int slices) {
  __shared__ float part[32][33];
  chain_point();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane, which = blockIdx.y;
  float* out = which ? a.db : a.dw;
  if (!out) return;
  float s = 0.f;
  if (c < a.cols) {
#pragma unroll 4
    for (int i = warp; i < slices; i += 32) s += a.work[(static_cast<long long>(i) * 2 + which) * a.cols + c];
  }
  part[lane][warp] = s;
  __syncthreads();
  s = warp_sum(part[warp][lane]);         // the warps' sums of column `warp`
  const int col = blockIdx.x * 32 + warp;
  if (lane == 0 && col < a.cols) out[col] = a.add ? out[col] + s : s;
}

bool ln_fits(const AerisLayerNorm* a) {
  return a->rows > 0 && a->rows <= 0x7fffffff && a->cols > 0 && a->x && a->y && a->stats && a->ld_x >= 0 && a->ld_y >= a->cols &&
         (reinterpret_cast<uintptr_t>(a->stats) & 7) == 0;       // read and written as float2
}

}  // namespace

}  // namespace aeris

#include "layer_norm_fast.cuh"

using namespace aeris;

extern "C" int aeris_layer_norm_fwd(const AerisLayerNorm* a, void* stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (!ln_fits(a)) return -1;
  int r = a->f32 ? ln_fwd_fast<float>(*a, stream) : ln_fwd_fast<__nv_bfloat16>(*a, stream);
  if (r <= 0) return r ? r : 1;
  const dim3 grid(static_cast<unsigned>(a->rows));
  r = a->f32 ? launch_chained(ln_fwd_any_kernel<float>, grid, LN_THREADS, 0, stream, *a)
             : launch_chained(ln_fwd_any_kernel<__nv_bfloat16>, grid, LN_THREADS, 0, stream, *a);
  return r ? r : 1;
}

extern "C" int aeris_layer_norm_bwd(const AerisLayerNorm* a, void* stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (!ln_fits(a) || !a->dy || a->ld_dy < 0) return -1;
  const bool sums = a->dw || a->db;
  if (sums && (a->slices <= 0 || a->slices > 65535 || (a->slices > 1) != (a->work != nullptr))) return -2;
  if (sums && !a->work && a->cols > 4096) return -3;       // a CTA's column sums are in shared memory
  int n = 1, slices = a->slices;
  int r = a->f32 ? ln_bwd_fast<float>(*a, stream, slices) : ln_bwd_fast<__nv_bfloat16>(*a, stream, slices);
  if (r < 0) return r;
  const bool fast = r == 0;
  if (!fast && sums) {     // first: the gradient of x may take the place of x or dy
    const dim3 grid((a->cols + LN_COLS - 1) / LN_COLS, a->slices);
    r = a->f32 ? launch_chained(ln_sums_any_kernel<float>, grid, LN_THREADS, 0, stream, *a)
               : launch_chained(ln_sums_any_kernel<__nv_bfloat16>, grid, LN_THREADS, 0, stream, *a);
    if (r) return r;
    ++n;
  }
  if (sums && a->work) {
    r = launch_chained(ln_join_kernel, dim3((a->cols + 31) / 32, 2), 1024, 0, stream, *a, slices);
    if (r) return r;
    ++n;
  }
  if (fast) return n;
  const dim3 grid(static_cast<unsigned>(a->rows));
  r = a->f32 ? launch_chained(ln_bwd_any_kernel<float>, grid, LN_THREADS, 0, stream, *a)
             : launch_chained(ln_bwd_any_kernel<__nv_bfloat16>, grid, LN_THREADS, 0, stream, *a);
  return r ? r : n;
}
