// RMS norms of queries and keys over each head's channels, with the position rotation in the same pass, and its gradients.
//
//   forward    z = w * x * r, r = (mean(x^2) + eps)^-1/2 over the head's d channels; y = R z, where R turns the channel pair
//              (2i, 2i + 1) by the angle of table row `pos` (i < rot / 2; channels from rot on are left as they are)
//   backward   dz = R^T dy; dw = sum over rows and heads of dz * x * r; with g = dz * w:
//              dx = r * (g - x r * mean(g x r))
//
// Both are bound by memory: 4 bytes of bf16 traffic an element forward, 6 backward, for about ten operations. A group of lanes
// (the power of two that holds d / 8) owns one head of a row at a time, eight channels to a lane, so that a head is one
// 16-byte load a lane, its sum of squares a few shuffles, and a pair to be turned lies in one lane. A row's heads are cut into
// parts of q or of k alone, as few as fill the GPU, one step each where rows are few (single tokens); a block stays with its part
// and its warps walk over rows, so that a lane's weights, and in the backward pass its sums for dw, are one set of eight
// registers, strides are uniform, and angles are read once a row. Everything between load and store is fp32.
#include "api.h"
#include "common.cuh"
#include "host.h"

namespace aeris {

constexpr int QKN_THREADS = 256;
constexpr int QKN_WARPS = QKN_THREADS / 32;
constexpr int QKN_MAX_D = 256;

// Eight values of one head in a lane: with VEC the channels 8 i .. 8 i + 7 of lane i, from one or two 16-byte loads at the lane's
// own address; else (any even width, any alignment) the pairs lane, lane + 32, .. of the whole warp from the head's start on.
template <typename T, bool VEC> struct HeadRaw;
template <> struct HeadRaw<__nv_bfloat16, true> {
  uint4 a;
  __device__ void load(const __nv_bfloat16* p, bool mine, int, int) {
    a = make_uint4(0, 0, 0, 0);
    if (mine) a = *reinterpret_cast<const uint4*>(p);
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
  static __device__ void store(__nv_bfloat16* p, bool mine, int, int, const float (&v)[8]) {
    if (mine)
      *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]),
                                                        pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
  }
};
template <> struct HeadRaw<float, true> {
  float4 a, b;
  __device__ void load(const float* p, bool mine, int, int) {
    a = b = make_float4(0.f, 0.f, 0.f, 0.f);
    if (mine) {
      a = *reinterpret_cast<const float4*>(p);
      b = *reinterpret_cast<const float4*>(p + 4);
    }
  }
  __device__ void get(float (&v)[8]) const {
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
  static __device__ void store(float* p, bool mine, int, int, const float (&v)[8]) {
    if (mine) {
      *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
      *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
    }
  }
};
__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void from_float(float x, float* p) { *p = x; }
__device__ __forceinline__ void from_float(float x, __nv_bfloat16* p) { *p = __float2bfloat16_rn(x); }
template <typename T> struct HeadRaw<T, false> {
  float f[8];
  __device__ void load(const T* p, bool mine, int lane, int d) {
    if (!mine) d = 0;
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
  static __device__ void store(T* p, bool mine, int lane, int d, const float (&v)[8]) {
    if (!mine) d = 0;
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

// What a block works on: `steps` steps of 32 / group heads of q or k, from head `first` on; its warps take rows `row`, row +
// stride, ..
struct Part {
  int lane, i, sub, per_step, first, steps, heads;
  bool is_k;
  int row, stride;
  __device__ Part(const AerisQkNorm& a, int group, int part_steps) {
    lane = threadIdx.x & 31;
    i = lane & (group - 1);
    sub = lane / group;
    per_step = 32 / group;
    const int q_steps = (a.heads + per_step - 1) / per_step, k_steps = (a.kv_heads + per_step - 1) / per_step;
    const int q_parts = (q_steps + part_steps - 1) / part_steps, parts = q_parts + (k_steps + part_steps - 1) / part_steps;
    const int part = blockIdx.x % parts;                // the grid is a multiple of the parts
    is_k = part >= q_parts;
    heads = is_k ? a.kv_heads : a.heads;
    const int step = (is_k ? part - q_parts : part) * part_steps;
    steps = min(part_steps, (is_k ? k_steps : q_steps) - step);
    first = step * per_step;
    row = blockIdx.x / parts * QKN_WARPS + (threadIdx.x >> 5);
    stride = gridDim.x / parts * QKN_WARPS;
  }
};
template <typename T, bool VEC> __device__ __forceinline__ T* lane_start(const AerisHeads& t, const Part& w) {
  return reinterpret_cast<T*>(const_cast<void*>(t.ptr)) + w.row * t.row + (w.first + w.sub) * t.head + (VEC ? 8 * w.i : 0);
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(QKN_THREADS, VEC ? 4 : 2) qk_norm_fwd_kernel(const AerisQkNorm a, int group, int part_steps) {
  constexpr int U = 3;                        // heads in flight per lane
  const Part t(a, group, part_steps);
  const AerisHeads in = t.is_k ? a.k : a.q, out = t.is_k ? a.k_out : a.q_out;
  const T* x_row = lane_start<const T, VEC>(in, t);
  T* y_row = lane_start<T, VEC>(out, t);
  const float inv_d = 1.f / a.d;
  const int heads = VEC && 8 * t.i >= a.d ? 0 : t.heads - t.first - t.sub;      // of the lane's, from its first one on
  chain_point();
  float w[8];
  load_weight<VEC>(t.is_k ? a.wk : a.wq, a.w_bf16, t.i, a.d, w);
  for (int row = t.row; row < a.rows; row += t.stride, x_row += t.stride * in.row, y_row += t.stride * out.row) {
    float c[4], s[4];
    const long long at = a.rot ? table_row(a, row) : 0;
    if (at < 0) continue;
    load_angles<VEC>(a, at, t.i, c, s);
    const T* x = x_row;
    T* y = y_row;
#pragma unroll 1
    for (int step = 0; step < t.steps; step += U) {
      HeadRaw<T, VEC> raw[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        raw[u].load(x + u * (t.per_step * in.head), step + u < t.steps && (step + u) * t.per_step < heads, t.i, a.d);
      x += U * (t.per_step * in.head);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (step + u >= t.steps) break;
        float v[8];
        raw[u].get(v);
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
        HeadRaw<T, VEC>::store(y + u * (t.per_step * out.head), (step + u) * t.per_step < heads, t.i, a.d, v);
      }
      y += U * (t.per_step * out.head);
    }
  }
}

// The sums for dw stay in a lane's registers over all rows; a block adds up its warps' in shared memory and writes one row
// [d] of `sums`, which qk_norm_sums_kernel adds up in a fixed order: no atomics, the same bits on every run.
template <typename T, bool VEC>
__global__ void __launch_bounds__(QKN_THREADS, 2) qk_norm_bwd_kernel(const AerisQkNorm a, int group, int part_steps) {
  constexpr int U = 2;
  __shared__ float red[QKN_WARPS][QKN_MAX_D];
  const Part t(a, group, part_steps);
  const AerisHeads in = t.is_k ? a.k : a.q, grad = t.is_k ? a.dk : a.dq, out = t.is_k ? a.k_out : a.q_out;
  const T *x_row = lane_start<const T, VEC>(in, t), *dy_row = lane_start<const T, VEC>(grad, t);
  T* dx_row = lane_start<T, VEC>(out, t);
  const float inv_d = 1.f / a.d;
  const int heads = VEC && 8 * t.i >= a.d ? 0 : t.heads - t.first - t.sub;
  chain_point();
  float w[8], dw[8];
  load_weight<VEC>(t.is_k ? a.wk : a.wq, a.w_bf16, t.i, a.d, w);
#pragma unroll
  for (int j = 0; j < 8; ++j) dw[j] = 0.f;
  for (int row = t.row; row < a.rows;
       row += t.stride, x_row += t.stride * in.row, dy_row += t.stride * grad.row, dx_row += t.stride * out.row) {
    float c[4], s[4];
    const long long at = a.rot ? table_row(a, row) : 0;
    if (at < 0) continue;
    load_angles<VEC>(a, at, t.i, c, s);
    const T *x = x_row, *dy = dy_row;
    T* dx = dx_row;
#pragma unroll 1
    for (int step = 0; step < t.steps; step += U) {
      HeadRaw<T, VEC> rx[U], rg[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const bool mine = step + u < t.steps && (step + u) * t.per_step < heads;
        rx[u].load(x + u * (t.per_step * in.head), mine, t.i, a.d);
        rg[u].load(dy + u * (t.per_step * grad.head), mine, t.i, a.d);
      }
      x += U * (t.per_step * in.head);
      dy += U * (t.per_step * grad.head);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (step + u >= t.steps) break;
        float v[8], g[8];
        rx[u].get(v);
        rg[u].get(g);
        float ss = 0.f, dot = 0.f;
        // mean(g x r) needs no r before its sum: both sums go through the shuffles together
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float e = g[2 * j] * c[j] + g[2 * j + 1] * s[j], o = g[2 * j + 1] * c[j] - g[2 * j] * s[j];
          ss += v[2 * j] * v[2 * j] + v[2 * j + 1] * v[2 * j + 1];
          g[2 * j] = e;
          g[2 * j + 1] = o;
          dot += e * w[2 * j] * v[2 * j] + o * w[2 * j + 1] * v[2 * j + 1];
        }
        for (int o = group >> 1; o > 0; o >>= 1) {
          ss += __shfl_xor_sync(0xffffffffu, ss, o);
          dot += __shfl_xor_sync(0xffffffffu, dot, o);
        }
        const float r = rsqrtf(ss * inv_d + a.eps), m = dot * inv_d * r;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float xhat = v[j] * r;
          dw[j] += g[j] * xhat;
          g[j] = r * (g[j] * w[j] - xhat * m);
        }
        HeadRaw<T, VEC>::store(dx + u * (t.per_step * out.head), (step + u) * t.per_step < heads, t.i, a.d, g);
      }
      dx += U * (t.per_step * out.head);
    }
  }
  const int warp = threadIdx.x >> 5;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    for (int o = group; o < 32; o <<= 1) dw[j] += __shfl_xor_sync(0xffffffffu, dw[j], o);
    const int e = pair_channel<VEC>(t.i, j / 2) + (j & 1);
    if (t.sub == 0 && e < a.d) red[warp][e] = dw[j];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < a.d; e += QKN_THREADS) {
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < QKN_WARPS; ++k) sum += red[k][e];
    a.sums[static_cast<long long>(blockIdx.x) * a.d + e] = sum;
  }
}

// dw from one row of sums per block, of which `q_parts` of every `parts` belong to q: 32 channels of q (blockIdx.y = 0) or k per
// block, one warp's lanes side by side, 32 warps over the rows.
__global__ void __launch_bounds__(1024) qk_norm_sums_kernel(const float* __restrict__ sums, int blocks, int parts, int q_parts, int d,
                                                            float* dwq, float* dwk, int add) {
  __shared__ float red[32][33];
  chain_point();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t = blockIdx.x * 32 + lane;
  const int first = blockIdx.y ? q_parts : 0, mine = blockIdx.y ? parts - q_parts : q_parts, n = blocks / parts * mine;
  float v = 0.f;
  if (t < d)
    for (int r = warp; r < n; r += 32) v += sums[(r / mine * parts + first + r % mine) * static_cast<long long>(d) + t];
  red[warp][lane] = v;
  __syncthreads();
  v = red[lane][warp];
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int at = blockIdx.x * 32 + warp;
  if (lane == 0 && at < d) {
    float* p = (blockIdx.y ? dwk : dwq) + at;
    *p = v + (add ? *p : 0.f);
  }
}

namespace {

bool vectors(const AerisHeads& t, int size) {
  return (reinterpret_cast<uintptr_t>(t.ptr) % 16 == 0) && (t.row * size) % 16 == 0 && (t.head * size) % 16 == 0;
}

// Lanes per head, steps per part and blocks. Parts of q and k are about as long as one another (a part has at most the steps of
// the one with fewer heads), and shorter where there would be fewer blocks than fit.
struct Shape {
  int group, part_steps, parts, q_parts, grid;
};
Shape shape_of(const AerisQkNorm& a, bool vec, int blocks_per_sm, int most) {
  Shape s;
  s.group = 32;
  if (vec)
    for (s.group = 1; 8 * s.group < a.d;) s.group *= 2;
  const int per = 32 / s.group, q = (a.heads + per - 1) / per, k = (a.kv_heads + per - 1) / per;
  int cap = num_sms() * blocks_per_sm;
  if (cap > most) cap = most;
  const long long row_blocks = (a.rows + QKN_WARPS - 1) / QKN_WARPS;
  const int few = (q + k + 127) / 128;        // at most so many parts, whatever the number of heads
  s.part_steps = q < k ? q : k;
  if (s.part_steps < few) s.part_steps = few;
  auto parts = [&](int n) { return (q + n - 1) / n + (k + n - 1) / n; };
  while (s.part_steps > few && row_blocks * parts(s.part_steps) < cap) --s.part_steps;
  s.parts = parts(s.part_steps);
  s.q_parts = (q + s.part_steps - 1) / s.part_steps;
  const long long by_rows = cap / s.parts;    // blocks of one part
  s.grid = s.parts * static_cast<int>(row_blocks < by_rows ? row_blocks : by_rows < 1 ? 1 : by_rows);
  return s;
}

int refused(const AerisQkNorm& a) {
  if (a.rows <= 0 || a.rows > 0x7fffffff - (1 << 20) || a.heads <= 0 || a.kv_heads <= 0 || a.d <= 0 || a.d % 2 || a.d > QKN_MAX_D) return -1;
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
  const Shape s = shape_of(a, vec, vec ? 4 : 2, 1 << 30);
  auto kern = a.f32 ? (vec ? qk_norm_fwd_kernel<float, true> : qk_norm_fwd_kernel<float, false>)
                    : (vec ? qk_norm_fwd_kernel<__nv_bfloat16, true> : qk_norm_fwd_kernel<__nv_bfloat16, false>);
  return launch_chained(kern, s.grid, QKN_THREADS, 0, stream, a, s.group, s.part_steps);
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
  const Shape s = shape_of(a, vec, 2, a.sum_rows);
  if (s.grid > a.sum_rows) return -5;
  auto kern = a.f32 ? (vec ? qk_norm_bwd_kernel<float, true> : qk_norm_bwd_kernel<float, false>)
                    : (vec ? qk_norm_bwd_kernel<__nv_bfloat16, true> : qk_norm_bwd_kernel<__nv_bfloat16, false>);
  if (const int rc = launch_chained(kern, s.grid, QKN_THREADS, 0, stream, a, s.group, s.part_steps)) return rc;
  if (const int rc = launch_chained(qk_norm_sums_kernel, dim3((a.d + 31) / 32, 2), 1024, 0, stream, a.sums, s.grid, s.parts,
                                    s.q_parts, a.d, a.dwq, a.dwk, a.add_dw))
    return rc;
  return 2;
}
