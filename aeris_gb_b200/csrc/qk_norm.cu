// RMS norms of queries and keys over each head's channels, with the position rotation in the same pass, and its gradients.
//
//   forward    z = w * x * r, r = (mean(x^2) + eps)^-1/2 over the head's d channels; y = R z, where R turns the channel pair
//              (2i, 2i + 1) by the angle of table row `pos` (i < rot / 2; channels from rot on are left as they are)
//   backward   dz = R^T dy; dw = sum over rows and heads of dz * x * r; with g = dz * w:
//              dx = r * (g - x r * mean(g x r))
//
// Both are bound by memory: 4 bytes of bf16 traffic an element forward, 6 backward, for about ten operations. A group of lanes
// (the power of two that holds d / 8) owns one head of a row at a time, eight channels to a lane, so that a head is one
// 16-byte load a lane, its sum of squares a few shuffles, and a pair to be turned lies in one lane. A warp walks over the
// heads of one row: a lane's weights stay in registers for the whole kernel and its angles for the row. Where rows are few
// (single tokens) the heads of a row are split over several warps instead. Everything between load and store is fp32.
#include "api.h"
#include "common.cuh"
#include "host.h"

namespace aeris {

constexpr int QKN_THREADS = 256;
constexpr int QKN_WARPS = QKN_THREADS / 32;
constexpr int QKN_MAX_D = 256;

// Eight values of one head in a lane: with VEC the channels 8 i .. 8 i + 7 of lane i, from one or two 16-byte loads; else
// (any even width, any alignment) the pairs lane, lane + 32, .. of the whole warp.
template <typename T, bool VEC> struct HeadRaw;
template <> struct HeadRaw<__nv_bfloat16, true> {
  uint4 a;
  __device__ void load(const __nv_bfloat16* p, int i, int d) {
    a = make_uint4(0, 0, 0, 0);
    if (8 * i < d) a = *reinterpret_cast<const uint4*>(p + 8 * i);
  }
  __device__ void get(float (&v)[8]) const {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = unpack_bf16x2(w[j]);
      v[2 * j] = f.x;
      v[2 * j + 1] = f.y;
    }
  }
  static __device__ void store(__nv_bfloat16* p, int i, int d, const float (&v)[8]) {
    if (8 * i < d)
      *reinterpret_cast<uint4*>(p + 8 * i) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]),
                                                        pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
  }
};
template <> struct HeadRaw<float, true> {
  float4 a, b;
  __device__ void load(const float* p, int i, int d) {
    a = b = make_float4(0.f, 0.f, 0.f, 0.f);
    if (8 * i < d) {
      a = *reinterpret_cast<const float4*>(p + 8 * i);
      b = *reinterpret_cast<const float4*>(p + 8 * i + 4);
    }
  }
  __device__ void get(float (&v)[8]) const {
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
  static __device__ void store(float* p, int i, int d, const float (&v)[8]) {
    if (8 * i < d) {
      *reinterpret_cast<float4*>(p + 8 * i) = make_float4(v[0], v[1], v[2], v[3]);
      *reinterpret_cast<float4*>(p + 8 * i + 4) = make_float4(v[4], v[5], v[6], v[7]);
    }
  }
};
__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void from_float(float x, float* p) { *p = x; }
__device__ __forceinline__ void from_float(float x, __nv_bfloat16* p) { *p = __float2bfloat16_rn(x); }
template <typename T> struct HeadRaw<T, false> {
  float f[8];
  __device__ void load(const T* p, int lane, int d) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int e = 2 * (j * 32 + lane);
      f[2 * j] = e < d ? to_float(p[e]) : 0.f;
      f[2 * j + 1] = e < d ? to_float(p[e + 1]) : 0.f;
    }
  }
  __device__ void get(float (&v)[8]) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = f[j];
  }
  static __device__ void store(T* p, int lane, int d, const float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int e = 2 * (j * 32 + lane);
      if (e < d) {
        from_float(v[2 * j], p + e);
        from_float(v[2 * j + 1], p + e + 1);
      }
    }
  }
};

// First channel of the lane's pair j.
template <bool VEC> __device__ __forceinline__ int pair_channel(int i, int j) { return VEC ? 8 * i + 2 * j : 2 * (j * 32 + i); }

template <bool VEC>
__device__ __forceinline__ void load_weight(const void* w, int bf16, int i, int d, float (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int e = pair_channel<VEC>(i, j / 2) + (j & 1);
    v[j] = e >= d ? 0.f : bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(w)[e])
                               : reinterpret_cast<const float*>(w)[e];
  }
}

// Row of the table for `row`, or -1 where its position lies outside (recorded in the status word).
__device__ __forceinline__ long long table_row(const AerisQkNorm& a, long long row) {
  if (!a.pos) return row % a.L;
  const long long p = a.pos64 ? reinterpret_cast<const long long*>(a.pos)[row] : reinterpret_cast<const int*>(a.pos)[row];
  if (p >= 0 && p < a.L) return p;
  atomicCAS(a.status, 0, ERR_BOUNDS);
  return -1;
}

template <bool VEC>
__device__ __forceinline__ void load_angles(const AerisQkNorm& a, long long at, int i, float (&c)[4], float (&s)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    c[j] = 1.f;
    s[j] = 0.f;
  }
  if (VEC) {                                  // rot is a multiple of 8 here: a lane turns all its pairs or none
    if (8 * i < a.rot) {
      const float4 x = *reinterpret_cast<const float4*>(a.cos + at * (a.rot / 2) + 4 * i);
      const float4 y = *reinterpret_cast<const float4*>(a.sin + at * (a.rot / 2) + 4 * i);
      c[0] = x.x; c[1] = x.y; c[2] = x.z; c[3] = x.w;
      s[0] = y.x; s[1] = y.y; s[2] = y.z; s[3] = y.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int p = j * 32 + i;
      if (p < a.rot / 2) {
        c[j] = a.cos[at * (a.rot / 2) + p];
        s[j] = a.sin[at * (a.rot / 2) + p];
      }
    }
  }
}

__device__ __forceinline__ float group_sum(float v, int group) {
  for (int o = group >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(QKN_THREADS) qk_norm_fwd_kernel(const AerisQkNorm a, int group, int parts) {
  constexpr int U = 4;                        // heads in flight per lane
  chain_point();
  const int lane = threadIdx.x & 31, i = lane & (group - 1), sub = lane / group, heads_per_step = 32 / group;
  const int q_steps = (a.heads + heads_per_step - 1) / heads_per_step;
  const int steps = q_steps + (a.kv_heads + heads_per_step - 1) / heads_per_step;
  const int per_part = (steps + parts - 1) / parts;
  const float inv_d = 1.f / a.d;
  float wq[8], wk[8];
  load_weight<VEC>(a.wq, a.w_bf16, i, a.d, wq);
  load_weight<VEC>(a.wk, a.w_bf16, i, a.d, wk);
  const long long units = a.rows * parts;
  for (long long u = blockIdx.x * static_cast<long long>(QKN_WARPS) + (threadIdx.x >> 5); u < units;
       u += static_cast<long long>(gridDim.x) * QKN_WARPS) {
    const long long row = parts == 1 ? u : u / parts;
    const int s0 = static_cast<int>(u - row * parts) * per_part, s1 = min(steps, s0 + per_part);
    float c[4], s[4];
    const long long at = a.rot ? table_row(a, row) : 0;
    if (at < 0) continue;
    load_angles<VEC>(a, at, i, c, s);
    auto section = [&](const AerisHeads& in, const AerisHeads& out, const float (&w)[8], int n, int first, int last) {
      const T* x = reinterpret_cast<const T*>(in.ptr) + row * in.row;
      T* y = reinterpret_cast<T*>(const_cast<void*>(out.ptr)) + row * out.row;
#pragma unroll 1
      for (int step = first; step < last; step += U) {
        HeadRaw<T, VEC> raw[U];
#pragma unroll
        for (int t = 0; t < U; ++t) {
          const int h = (step + t) * heads_per_step + sub;
          raw[t].load(x + h * in.head, i, step + t < last && h < n ? a.d : 0);
        }
#pragma unroll
        for (int t = 0; t < U; ++t) {
          if (step + t >= last) break;
          const int h = (step + t) * heads_per_step + sub;
          float v[8];
          raw[t].get(v);
          float ss = 0.f;
#pragma unroll
          for (int j = 0; j < 8; ++j) ss += v[j] * v[j];
          const float r = rsqrtf(group_sum(ss, group) * inv_d + a.eps);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float e = v[2 * j] * r * w[2 * j], o = v[2 * j + 1] * r * w[2 * j + 1];
            v[2 * j] = e * c[j] - o * s[j];
            v[2 * j + 1] = o * c[j] + e * s[j];
          }
          HeadRaw<T, VEC>::store(y + h * out.head, i, h < n ? a.d : 0, v);
        }
      }
    };
    if (s0 < q_steps) section(a.q, a.q_out, wq, a.heads, s0, min(s1, q_steps));
    if (s1 > q_steps) section(a.k, a.k_out, wk, a.kv_heads, max(s0, q_steps) - q_steps, s1 - q_steps);
  }
}

// The sums for dw stay in a lane's registers over all rows; a block adds up its warps' in shared memory and writes one row
// [2][d] of `sums`, which qk_norm_sums_kernel adds up in a fixed order: no atomics, the same bits on every run. A single
// block writes the result itself.
template <typename T, bool VEC>
__global__ void __launch_bounds__(QKN_THREADS) qk_norm_bwd_kernel(const AerisQkNorm a, int group, int parts) {
  constexpr int U = 2;
  __shared__ float red[QKN_WARPS][2][QKN_MAX_D];
  chain_point();
  const int lane = threadIdx.x & 31, i = lane & (group - 1), sub = lane / group, heads_per_step = 32 / group;
  const int q_steps = (a.heads + heads_per_step - 1) / heads_per_step;
  const int steps = q_steps + (a.kv_heads + heads_per_step - 1) / heads_per_step;
  const int per_part = (steps + parts - 1) / parts;
  const float inv_d = 1.f / a.d;
  float wq[8], wk[8], dwq[8], dwk[8];
  load_weight<VEC>(a.wq, a.w_bf16, i, a.d, wq);
  load_weight<VEC>(a.wk, a.w_bf16, i, a.d, wk);
#pragma unroll
  for (int j = 0; j < 8; ++j) dwq[j] = dwk[j] = 0.f;
  const long long units = a.rows * parts;
  for (long long u = blockIdx.x * static_cast<long long>(QKN_WARPS) + (threadIdx.x >> 5); u < units;
       u += static_cast<long long>(gridDim.x) * QKN_WARPS) {
    const long long row = parts == 1 ? u : u / parts;
    const int s0 = static_cast<int>(u - row * parts) * per_part, s1 = min(steps, s0 + per_part);
    float c[4], s[4];
    const long long at = a.rot ? table_row(a, row) : 0;
    if (at < 0) continue;
    load_angles<VEC>(a, at, i, c, s);
    auto section = [&](const AerisHeads& in, const AerisHeads& grad, const AerisHeads& out, const float (&w)[8],
                       float (&dw)[8], int n, int first, int last) {
      const T* x = reinterpret_cast<const T*>(in.ptr) + row * in.row;
      const T* dy = reinterpret_cast<const T*>(grad.ptr) + row * grad.row;
      T* dx = reinterpret_cast<T*>(const_cast<void*>(out.ptr)) + row * out.row;
#pragma unroll 1
      for (int step = first; step < last; step += U) {
        HeadRaw<T, VEC> rx[U], rg[U];
#pragma unroll
        for (int t = 0; t < U; ++t) {
          const int h = (step + t) * heads_per_step + sub, d = step + t < last && h < n ? a.d : 0;
          rx[t].load(x + h * in.head, i, d);
          rg[t].load(dy + h * grad.head, i, d);
        }
#pragma unroll
        for (int t = 0; t < U; ++t) {
          if (step + t >= last) break;
          const int h = (step + t) * heads_per_step + sub;
          float v[8], g[8];
          rx[t].get(v);
          rg[t].get(g);
          float ss = 0.f;
#pragma unroll
          for (int j = 0; j < 8; ++j) ss += v[j] * v[j];
          const float r = rsqrtf(group_sum(ss, group) * inv_d + a.eps);
          float dot = 0.f;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float e = g[2 * j] * c[j] + g[2 * j + 1] * s[j], o = g[2 * j + 1] * c[j] - g[2 * j] * s[j];
            v[2 * j] *= r;
            v[2 * j + 1] *= r;
            dw[2 * j] += e * v[2 * j];
            dw[2 * j + 1] += o * v[2 * j + 1];
            g[2 * j] = e * w[2 * j];
            g[2 * j + 1] = o * w[2 * j + 1];
            dot += g[2 * j] * v[2 * j] + g[2 * j + 1] * v[2 * j + 1];
          }
          const float m = group_sum(dot, group) * inv_d;
#pragma unroll
          for (int j = 0; j < 8; ++j) g[j] = r * (g[j] - v[j] * m);
          HeadRaw<T, VEC>::store(dx + h * out.head, i, h < n ? a.d : 0, g);
        }
      }
    };
    if (s0 < q_steps) section(a.q, a.dq, a.q_out, wq, dwq, a.heads, s0, min(s1, q_steps));
    if (s1 > q_steps) section(a.k, a.dk, a.k_out, wk, dwk, a.kv_heads, max(s0, q_steps) - q_steps, s1 - q_steps);
  }
  const int warp = threadIdx.x >> 5;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    for (int o = group; o < 32; o <<= 1) {
      dwq[j] += __shfl_xor_sync(0xffffffffu, dwq[j], o);
      dwk[j] += __shfl_xor_sync(0xffffffffu, dwk[j], o);
    }
    const int e = pair_channel<VEC>(i, j / 2) + (j & 1);
    if (sub == 0 && e < a.d) {
      red[warp][0][e] = dwq[j];
      red[warp][1][e] = dwk[j];
    }
  }
  __syncthreads();
  for (int t = threadIdx.x; t < 2 * a.d; t += QKN_THREADS) {
    const int which = t >= a.d, e = t - which * a.d;
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < QKN_WARPS; ++k) sum += red[k][which][e];
    if (gridDim.x == 1) {
      float* dw = which ? a.dwk : a.dwq;
      dw[e] = sum + (a.add_dw ? dw[e] : 0.f);
    } else {
      a.sums[blockIdx.x * 2ll * a.d + t] = sum;
    }
  }
}

// dw[2][d] from `n` rows of sums: 32 channels per block, one warp's lanes side by side, 32 warps over the rows.
__global__ void __launch_bounds__(1024) qk_norm_sums_kernel(const float* __restrict__ sums, int n, int d, float* dwq,
                                                            float* dwk, int add) {
  __shared__ float red[32][33];
  chain_point();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t = blockIdx.x * 32 + lane;
  float v = 0.f;
  if (t < 2 * d)
    for (int r = warp; r < n; r += 32) v += sums[r * 2ll * d + t];
  red[warp][lane] = v;
  __syncthreads();
  v = red[lane][warp];
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int at = blockIdx.x * 32 + warp;
  if (lane == 0 && at < 2 * d) {
    float* p = at < d ? dwq + at : dwk + at - d;
    *p = v + (add ? *p : 0.f);
  }
}

namespace {

bool vectors(const AerisHeads& t, int size) {
  return (reinterpret_cast<uintptr_t>(t.ptr) % 16 == 0) && (t.row * size) % 16 == 0 && (t.head * size) % 16 == 0;
}

// Lanes per head, warps per row and blocks. A warp walks over a whole row unless that leaves multiprocessors idle.
struct Shape {
  bool vec;
  int group, parts, grid;
};
Shape shape_of(const AerisQkNorm& a, bool vec, int blocks_per_sm, int most) {
  Shape s;
  s.vec = vec;
  s.group = 32;
  if (vec)
    for (s.group = 1; 8 * s.group < a.d;) s.group *= 2;
  const int per = 32 / s.group, steps = (a.heads + per - 1) / per + (a.kv_heads + per - 1) / per;
  const long long warps = static_cast<long long>(num_sms()) * blocks_per_sm * QKN_WARPS;
  const long long parts = a.rows >= warps ? 1 : warps / a.rows;
  s.parts = static_cast<int>(parts < steps ? parts : steps);
  const long long blocks = (a.rows * s.parts + QKN_WARPS - 1) / QKN_WARPS;
  const long long cap = static_cast<long long>(num_sms()) * blocks_per_sm;
  s.grid = static_cast<int>(blocks < cap ? blocks : cap);
  if (s.grid > most) s.grid = most;
  return s;
}

int refused(const AerisQkNorm& a) {
  if (a.rows <= 0 || a.heads <= 0 || a.kv_heads <= 0 || a.d <= 0 || a.d % 2 || a.d > QKN_MAX_D) return -1;
  if (a.rot < 0 || a.rot % 2 || a.rot > a.d || (a.rot && (!a.cos || !a.sin || a.L <= 0)) || !a.wq || !a.wk) return -2;
  if (!a.q.ptr || !a.k.ptr || !a.q_out.ptr || !a.k_out.ptr || !a.status) return -3;
  return 0;
}

bool angles_in_vectors(const AerisQkNorm& a) {
  return !a.rot || (a.rot % 8 == 0 && reinterpret_cast<uintptr_t>(a.cos) % 16 == 0 && reinterpret_cast<uintptr_t>(a.sin) % 16 == 0);
}

}  // namespace
}  // namespace aeris

using namespace aeris;

extern "C" int aeris_qk_norm_fwd(const AerisQkNorm* p, void* stream_) {
  const AerisQkNorm& a = *p;
  if (const int rc = refused(a)) return rc;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  const int size = a.f32 ? 4 : 2;
  const bool vec = a.d % 8 == 0 && angles_in_vectors(a) && vectors(a.q, size) && vectors(a.k, size) && vectors(a.q_out, size) &&
                   vectors(a.k_out, size);
  const Shape s = shape_of(a, vec, 8, 1 << 30);
  auto kern = a.f32 ? (vec ? qk_norm_fwd_kernel<float, true> : qk_norm_fwd_kernel<float, false>)
                    : (vec ? qk_norm_fwd_kernel<__nv_bfloat16, true> : qk_norm_fwd_kernel<__nv_bfloat16, false>);
  return launch_chained(kern, s.grid, QKN_THREADS, 0, stream, a, s.group, s.parts);
}

// Returns the number of kernels launched, or a negative code.
extern "C" int aeris_qk_norm_bwd(const AerisQkNorm* p, void* stream_) {
  const AerisQkNorm& a = *p;
  if (const int rc = refused(a)) return rc;
  if (!a.dq.ptr || !a.dk.ptr || !a.dwq || !a.dwk || !a.sums || a.sum_rows <= 0) return -4;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  const int size = a.f32 ? 4 : 2;
  const bool vec = a.d % 8 == 0 && angles_in_vectors(a) && vectors(a.q, size) && vectors(a.k, size) && vectors(a.q_out, size) &&
                   vectors(a.k_out, size) && vectors(a.dq, size) && vectors(a.dk, size);
  const Shape s = shape_of(a, vec, 4, a.sum_rows);
  auto kern = a.f32 ? (vec ? qk_norm_bwd_kernel<float, true> : qk_norm_bwd_kernel<float, false>)
                    : (vec ? qk_norm_bwd_kernel<__nv_bfloat16, true> : qk_norm_bwd_kernel<__nv_bfloat16, false>);
  if (const int rc = launch_chained(kern, s.grid, QKN_THREADS, 0, stream, a, s.group, s.parts)) return rc;
  if (s.grid == 1) return 1;
  if (const int rc = launch_chained(qk_norm_sums_kernel, (2 * a.d + 31) / 32, 1024, 0, stream, a.sums, s.grid, a.d, a.dwq, a.dwk,
                                    a.add_dw))
    return rc;
  return 2;
}
