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
// parts of q or of k alone, one of each where rows fill the GPU, down to one step each where they are few (single tokens); a block
// stays with its part and its warps walk over rows, so that a lane's weights, and in the backward pass its sums for dw, are one
// set of eight registers, strides are uniform, and angles are read once a row. q and k have blocks in proportion to their
// heads. Everything between load and store is fp32. 64,800 rows of 24 + 24 heads of 64, bf16: forward 137 us, 5.8 TB/s (89 % of
// what a plain copy reaches); backward 212 us, 5.6 TB/s; 28,800 rows of 40 + 40 heads of 128 backward 316 us. One row, or one
// window of 900, takes the GPU 5 to 7 us, less than the host needs for the call (14).
#include "api.h"
#include "common.cuh"
#include "host.h"

namespace aeris {

constexpr int QKN_THREADS = 256;
constexpr int QKN_WARPS = QKN_THREADS / 32;
constexpr int QKN_MAX_D = 256;

// Eight values of one head in a lane as two-wide fp32 operands, half the instructions of single ones: the even and the odd
// channels of pairs 0 and 1 (e[0], o[0]) and of pairs 2 and 3 (e[1], o[1]), so that turning a pair swaps nothing.
struct Eight {
  uint64_t e[2], o[2];
};
__device__ __forceinline__ uint64_t f2_all(float x) { return f2_pack(x, x); }
__device__ __forceinline__ float f2_sum(uint64_t v) {
  float a, b;
  f2_unpack(v, a, b);
  return a + b;
}
__device__ __forceinline__ uint64_t f2_neg(uint64_t v) { return v ^ 0x8000000080000000ull; }

// With VEC a lane i has the channels 8 i .. 8 i + 7, from one or two 16-byte loads at the lane's own address; else (any even
// width, any alignment) the pairs lane, lane + 32, .. of the whole warp, from the head's start on.
template <typename T, bool VEC> struct HeadRaw;
template <> struct HeadRaw<__nv_bfloat16, true> {
  uint4 a;
  __device__ void load(const __nv_bfloat16* p, bool mine, int, int, int = 0) {
    a = make_uint4(0, 0, 0, 0);
    if (mine) a = *reinterpret_cast<const uint4*>(p);
  }
  __device__ Eight get() const {
    auto lo = [](uint32_t x) { return __uint_as_float(x << 16); };
    auto hi = [](uint32_t x) { return __uint_as_float(x & 0xffff0000u); };
    return {{f2_pack(lo(a.x), lo(a.y)), f2_pack(lo(a.z), lo(a.w))}, {f2_pack(hi(a.x), hi(a.y)), f2_pack(hi(a.z), hi(a.w))}};
  }
  static __device__ void store(__nv_bfloat16* p, bool mine, int, int, const Eight& v) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float e0, e1, o0, o1;
      f2_unpack(v.e[k], e0, e1);
      f2_unpack(v.o[k], o0, o1);
      w[2 * k] = pack_bf16x2(e0, o0);
      w[2 * k + 1] = pack_bf16x2(e1, o1);
    }
    if (mine) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <> struct HeadRaw<float, true> {
  float4 a, b;
  __device__ void load(const float* p, bool mine, int, int, int next = 4) {      // next: from one vector to the other
    a = b = make_float4(0.f, 0.f, 0.f, 0.f);
    if (mine) {
      a = *reinterpret_cast<const float4*>(p);
      b = *reinterpret_cast<const float4*>(p + next);
    }
  }
  __device__ Eight get() const { return {{f2_pack(a.x, a.z), f2_pack(b.x, b.z)}, {f2_pack(a.y, a.w), f2_pack(b.y, b.w)}}; }
  static __device__ void store(float* p, bool mine, int, int, const Eight& v) {
    float4 x, y;
    f2_unpack(v.e[0], x.x, x.z);
    f2_unpack(v.o[0], x.y, x.w);
    f2_unpack(v.e[1], y.x, y.z);
    f2_unpack(v.o[1], y.y, y.w);
    if (mine) {
      *reinterpret_cast<float4*>(p) = x;
      *reinterpret_cast<float4*>(p + 4) = y;
    }
  }
};
__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void from_float(float x, float* p) { *p = x; }
__device__ __forceinline__ void from_float(float x, __nv_bfloat16* p) { *p = __float2bfloat16_rn(x); }
__device__ __forceinline__ Eight eight_of(const float (&f)[8]) {
  return {{f2_pack(f[0], f[2]), f2_pack(f[4], f[6])}, {f2_pack(f[1], f[3]), f2_pack(f[5], f[7])}};
}
__device__ __forceinline__ void singles(const Eight& v, float (&f)[8]) {
  f2_unpack(v.e[0], f[0], f[2]);
  f2_unpack(v.o[0], f[1], f[3]);
  f2_unpack(v.e[1], f[4], f[6]);
  f2_unpack(v.o[1], f[5], f[7]);
}
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
  __device__ Eight get() const { return eight_of(f); }
  static __device__ void store(T* p, bool mine, int lane, int d, const Eight& x) {
    float v[8];
    singles(x, v);
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

template <bool VEC> __device__ __forceinline__ Eight load_weight(const void* w, int bf16, int i, int d) {
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int e = pair_channel<VEC>(i, j / 2) + (j & 1);
    v[j] = e >= d ? 0.f : bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(w)[e])
                               : reinterpret_cast<const float*>(w)[e];
  }
  return eight_of(v);
}

// Row of the table for `row`, or -1 where its position lies outside (recorded in the status word).
__device__ __forceinline__ int table_row(const AerisQkNorm& a, int row) {
  if (row >= a.rows || !a.rot) return 0;
  if (!a.pos) return row % a.L;
  const long long p = a.pos64 ? reinterpret_cast<const long long*>(a.pos)[row] : reinterpret_cast<const int*>(a.pos)[row];
  if (p >= 0 && p < a.L) return static_cast<int>(p);
  atomicCAS(a.status, 0, ERR_BOUNDS);
  return -1;
}

struct Angles {
  uint64_t c[2], s[2];                        // of pairs 0 and 1, of pairs 2 and 3
};
template <bool VEC> __device__ __forceinline__ Angles load_angles(const AerisQkNorm& a, int row, int i) {
  const long long at = row;
  float c[4], s[4];
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
  return {{f2_pack(c[0], c[1]), f2_pack(c[2], c[3])}, {f2_pack(s[0], s[1]), f2_pack(s[2], s[3])}};
}

__device__ __forceinline__ float group_sum(float v, int group) {
  for (int o = group >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// What a block works on: `steps` steps of 32 / group heads of q or k, from head `first` on; its warps take rows `row`, row +
// stride, ..
struct QkCut {
  int group, q_len, k_len, q_blocks, k_blocks;          // steps of a part, blocks of all parts of q and of k
};
struct Part {
  int lane, i, sub, per_step, first, steps, heads;
  bool is_k;
  int row, stride;
  __device__ Part(const AerisQkNorm& a, const QkCut& cut) {
    lane = threadIdx.x & 31;
    i = lane & (cut.group - 1);
    sub = lane / cut.group;
    per_step = 32 / cut.group;
    is_k = blockIdx.x >= cut.q_blocks;
    heads = is_k ? a.kv_heads : a.heads;
    const int len = is_k ? cut.k_len : cut.q_len, all = (heads + per_step - 1) / per_step, parts = (all + len - 1) / len;
    const int block = is_k ? blockIdx.x - cut.q_blocks : blockIdx.x;
    const int step = block % parts * len;
    steps = min(len, all - step);
    first = step * per_step;
    row = block / parts * QKN_WARPS + (threadIdx.x >> 5);
    stride = (is_k ? cut.k_blocks : cut.q_blocks) / parts * QKN_WARPS;      // the blocks are a multiple of the parts
  }
};
template <typename T, bool VEC> __device__ __forceinline__ T* lane_start(const AerisHeads& t, const Part& w) {
  return reinterpret_cast<T*>(const_cast<void*>(t.ptr)) + w.row * t.row + (w.first + w.sub) * t.head + (VEC ? 8 * w.i : 0);
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(QKN_THREADS, VEC ? 4 : 2) qk_norm_fwd_kernel(const AerisQkNorm a, const QkCut cut) {
  constexpr int U = 3;                        // heads in flight per lane
  const Part t(a, cut);
  const AerisHeads in = t.is_k ? a.k : a.q, out = t.is_k ? a.k_out : a.q_out;
  const T* x_row = lane_start<const T, VEC>(in, t);
  T* y_row = lane_start<T, VEC>(out, t);
  const float inv_d = 1.f / a.d;
  const int heads = VEC && 8 * t.i >= a.d ? 0 : t.heads - t.first - t.sub;      // of the lane's, from its first one on
  chain_point();
  const Eight w = load_weight<VEC>(t.is_k ? a.wk : a.wq, a.w_bf16, t.i, a.d);
  for (int row = t.row; row < a.rows; row += t.stride, x_row += t.stride * in.row, y_row += t.stride * out.row) {
    const int at = table_row(a, row);         // nothing but the angles waits for it
    const Angles r = load_angles<VEC>(a, max(at, 0), t.i);
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
        Eight v = raw[u].get();
        const uint64_t ss = f2_fma(v.o[1], v.o[1], f2_fma(v.e[1], v.e[1], f2_fma(v.o[0], v.o[0], f2_mul(v.e[0], v.e[0]))));
        const uint64_t scale = f2_all(rsqrtf(group_sum(f2_sum(ss), cut.group) * inv_d + a.eps));
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint64_t e = f2_mul(f2_mul(v.e[k], scale), w.e[k]), o = f2_mul(f2_mul(v.o[k], scale), w.o[k]);
          v.e[k] = f2_fma(e, r.c[k], f2_neg(f2_mul(o, r.s[k])));
          v.o[k] = f2_fma(o, r.c[k], f2_mul(e, r.s[k]));
        }
        HeadRaw<T, VEC>::store(y + u * (t.per_step * out.head), at >= 0 && (step + u) * t.per_step < heads, t.i, a.d, v);
      }
      y += U * (t.per_step * out.head);
    }
  }
}

// One head's gradient in a lane: v = x and g = dy on entry; dw is added to, g holds dx on return.
__device__ __forceinline__ void head_backward(const Eight& v, Eight& g, const Eight& w, const Angles& r, Eight& dw, int group,
                                              float inv_d, float eps) {
  uint64_t ss2 = 0, dot2 = 0;                 // two zeros
  Eight gw;
  // mean(g x r) needs no r before its sum: both sums go through the shuffles together
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const uint64_t e = f2_fma(g.e[k], r.c[k], f2_mul(g.o[k], r.s[k]));
    const uint64_t o = f2_fma(g.o[k], r.c[k], f2_neg(f2_mul(g.e[k], r.s[k])));
    g.e[k] = e;
    g.o[k] = o;
    gw.e[k] = f2_mul(e, w.e[k]);
    gw.o[k] = f2_mul(o, w.o[k]);
    ss2 = f2_fma(v.o[k], v.o[k], f2_fma(v.e[k], v.e[k], ss2));
    dot2 = f2_fma(gw.o[k], v.o[k], f2_fma(gw.e[k], v.e[k], dot2));
  }
  float ss = f2_sum(ss2), dot = f2_sum(dot2);
  for (int o = group >> 1; o > 0; o >>= 1) {
    ss += __shfl_xor_sync(0xffffffffu, ss, o);
    dot += __shfl_xor_sync(0xffffffffu, dot, o);
  }
  const float scale = rsqrtf(ss * inv_d + eps);
  const uint64_t s2 = f2_all(scale), m2 = f2_all(-dot * inv_d * scale * scale);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const uint64_t xe = f2_mul(v.e[k], s2), xo = f2_mul(v.o[k], s2);
    dw.e[k] = f2_fma(g.e[k], xe, dw.e[k]);
    dw.o[k] = f2_fma(g.o[k], xo, dw.o[k]);
    g.e[k] = f2_fma(xe, m2, f2_mul(gw.e[k], s2));
    g.o[k] = f2_fma(xo, m2, f2_mul(gw.o[k], s2));
  }
}

// The sums for dw stay in a lane's registers over all rows; a block adds up its warps' in shared memory and writes one row
// [d] of `sums`, which qk_norm_sums_kernel adds up in a fixed order: no atomics, the same bits on every run.
template <bool VEC>
__device__ __forceinline__ void block_sums(float (*red)[QKN_MAX_D], const Eight& sum8, const Part& t, int group, int d, float* sums) {
  const int warp = threadIdx.x >> 5;
  float dw[8];
  singles(sum8, dw);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    for (int o = group; o < 32; o <<= 1) dw[j] += __shfl_xor_sync(0xffffffffu, dw[j], o);
    const int e = pair_channel<VEC>(t.i, j / 2) + (j & 1);
    if (t.sub == 0 && e < d) red[warp][e] = dw[j];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < d; e += QKN_THREADS) {
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < QKN_WARPS; ++k) sum += red[k][e];
    sums[static_cast<long long>(blockIdx.x) * d + e] = sum;
  }
}

// Any even width, any alignment.
template <typename T>
__global__ void __launch_bounds__(QKN_THREADS, 2) qk_norm_bwd_kernel(const AerisQkNorm a, const QkCut cut) {
  __shared__ float red[QKN_WARPS][QKN_MAX_D];
  const Part t(a, cut);
  const AerisHeads in = t.is_k ? a.k : a.q, grad = t.is_k ? a.dk : a.dq, out = t.is_k ? a.k_out : a.q_out;
  const T *x = lane_start<const T, false>(in, t), *dy = lane_start<const T, false>(grad, t);
  T* dx = lane_start<T, false>(out, t);
  const float inv_d = 1.f / a.d;
  chain_point();
  const Eight w = load_weight<false>(t.is_k ? a.wk : a.wq, a.w_bf16, t.i, a.d);
  Eight dw = {};
  for (int row = t.row; row < a.rows; row += t.stride, x += t.stride * in.row, dy += t.stride * grad.row, dx += t.stride * out.row) {
    const int at = table_row(a, row);
    if (at < 0) continue;
    const Angles r = load_angles<false>(a, at, t.i);
#pragma unroll 1
    for (int step = 0; step < t.steps; ++step) {        // a head a step here
      HeadRaw<T, false> rx, rg;
      rx.load(x + step * in.head, true, t.i, a.d);
      rg.load(dy + step * grad.head, true, t.i, a.d);
      Eight g = rg.get();
      head_backward(rx.get(), g, w, r, dw, cut.group, inv_d, a.eps);
      HeadRaw<T, false>::store(dx + step * out.head, true, t.i, a.d, g);
    }
  }
  block_sums<false>(red, dw, t, cut.group, a.d, a.sums);
}

// Whole vectors. What a warp reads passes through a ring of its own in shared memory, a few steps ahead (asynchronous copies
// of 16 bytes that the same lane takes out again): with the loads in registers, two steps at a time, 127 registers left 16
// warps per SM too little under way (64,800 rows, 24 + 24 heads of 64: 265 us; ring 247, with two-wide arithmetic 212; three
// blocks an SM instead of two 217).
template <typename T>
__global__ void __launch_bounds__(QKN_THREADS, 2) qk_norm_bwd_ring_kernel(const AerisQkNorm a, const QkCut cut) {
  constexpr int VECS = sizeof(T) / 2, AHEAD = VECS == 1 ? 4 : 3;      // 16-byte vectors of eight values; stages of the ring
  __shared__ union {
    uint4 ring[QKN_WARPS][AHEAD][2][VECS][32];
    float red[QKN_WARPS][QKN_MAX_D];
  } sm;
  const Part t(a, cut);
  const AerisHeads in = t.is_k ? a.k : a.q, grad = t.is_k ? a.dk : a.dq, out = t.is_k ? a.k_out : a.q_out;
  const T *x = lane_start<const T, true>(in, t), *dy = lane_start<const T, true>(grad, t);      // of the copies ahead
  T* dx = lane_start<T, true>(out, t);
  const float inv_d = 1.f / a.d;
  const int heads = 8 * t.i >= a.d ? 0 : t.heads - t.first - t.sub;   // of the lane's, from its first one on
  uint4 (*ring)[2][VECS][32] = sm.ring[threadIdx.x >> 5];
  chain_point();
  const Eight w = load_weight<true>(t.is_k ? a.wk : a.wq, a.w_bf16, t.i, a.d);
  Eight dw = {};
  const long long in_step = t.per_step * in.head, grad_step = t.per_step * grad.head, out_step = t.per_step * out.head;
  int ahead_rows = t.row < a.rows ? (a.rows - 1 - t.row) / t.stride + 1 : 0, ahead_step = 0;
  uint32_t ahead_to = smem_u32(&ring[0][0][0][t.lane]);
  const uint32_t ring_end = ahead_to + AHEAD * sizeof(ring[0]);
  uint32_t from = ahead_to;
  auto next = [&](uint32_t slot) { return slot + sizeof(ring[0]) == ring_end ? ring_end - AHEAD * sizeof(ring[0]) : slot + sizeof(ring[0]); };
  auto copy = [&] {
    if (ahead_rows > 0) {
      if (ahead_step * t.per_step < heads) {
#pragma unroll
        for (int k = 0; k < VECS; ++k) {
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(ahead_to + 512 * k), "l"(x + 4 * k) : "memory");
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(ahead_to + 512 * (VECS + k)), "l"(dy + 4 * k) : "memory");
        }
      }
      x += in_step;
      dy += grad_step;
      if (++ahead_step == t.steps) {
        ahead_step = 0;
        --ahead_rows;
        x += t.stride * in.row - t.steps * in_step;
        dy += t.stride * grad.row - t.steps * grad_step;
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    ahead_to = next(ahead_to);
  };
#pragma unroll
  for (int k = 0; k < AHEAD - 1; ++k) copy();
  int next_at = table_row(a, t.row);
  for (int row = t.row; row < a.rows; row += t.stride, dx += t.stride * out.row - t.steps * out_step) {
    const int at = next_at;
    next_at = table_row(a, row + t.stride);
    const Angles r = load_angles<true>(a, at < 0 ? 0 : at, t.i);
#pragma unroll 1
    for (int step = 0; step < t.steps; ++step, dx += out_step) {
      copy();
      asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD - 1) : "memory");
      if (at >= 0) {
        const bool mine = step * t.per_step < heads;
        const T* slot = reinterpret_cast<const T*>(__cvta_shared_to_generic(from));
        constexpr int NEXT = 512 / sizeof(T);
        HeadRaw<T, true> rx, rg;
        rx.load(slot, mine, 0, 0, NEXT);
        rg.load(slot + VECS * NEXT, mine, 0, 0, NEXT);
        Eight g = rg.get();
        head_backward(rx.get(), g, w, r, dw, cut.group, inv_d, a.eps);
        HeadRaw<T, true>::store(dx, mine, 0, 0, g);
      }
      from = next(from);
    }
  }
  __syncthreads();                            // the ring becomes the sums' place
  block_sums<true>(sm.red, dw, t, cut.group, a.d, a.sums);
}

// dw from one row of sums per block, those of q before those of k: 32 channels of q (blockIdx.y = 0) or k per block, one warp's
// lanes side by side, 32 warps over the rows. A weight that q and k share has one sum of both (gridDim.y = 1, no rows of k).
__global__ void __launch_bounds__(1024) qk_norm_sums_kernel(const float* __restrict__ sums, int q_rows, int k_rows, int d, float* dwq,
                                                            float* dwk, int add) {
  __shared__ float red[32][33];
  chain_point();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t = blockIdx.x * 32 + lane;
  if (blockIdx.y) sums += static_cast<long long>(q_rows) * d;
  const int n = blockIdx.y ? k_rows : q_rows;
  float v = 0.f;
  if (t < d)
    for (int r = warp; r < n; r += 32) v += sums[r * static_cast<long long>(d) + t];
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

// Lanes per head, parts and blocks: `most` blocks in all, or the few that one row a warp and one step a part make. A row takes a
// warp as long as its rounds of `at_once` steps: by steps alone, two key heads next to ten of queries got a sixth of the blocks
// and took twice as long as those (12,345 rows of 72 channels, fp32: 27 us, by rounds 23).
QkCut cut_of(const AerisQkNorm& a, bool vec, int blocks_per_sm, int at_once, int most) {
  QkCut c;
  c.group = 32;
  if (vec)
    for (c.group = 1; 8 * c.group < a.d;) c.group *= 2;
  const int per = 32 / c.group, q = (a.heads + per - 1) / per, k = (a.kv_heads + per - 1) / per;
  int cap = num_sms() * blocks_per_sm;
  if (cap > most) cap = most;
  const long long row_blocks = (a.rows + QKN_WARPS - 1) / QKN_WARPS;
  auto side = [&](int steps, int share, int& len, int& blocks) {
    if (share < 1) share = 1;
    const long long want = (share + row_blocks - 1) / row_blocks;               // parts that fill the share
    const int parts = static_cast<int>(want < steps ? want : steps);
    len = (steps + parts - 1) / parts;
    const int real = (steps + len - 1) / len;
    const long long by_rows = share / real < 1 ? 1 : share / real;
    blocks = real * static_cast<int>(row_blocks < by_rows ? row_blocks : by_rows);
  };
  const int q_rounds = (q + at_once - 1) / at_once, k_rounds = (k + at_once - 1) / at_once;
  const int q_share = static_cast<int>(static_cast<long long>(cap) * q_rounds / (q_rounds + k_rounds));
  side(q, q_share, c.q_len, c.q_blocks);
  side(k, cap - q_share, c.k_len, c.k_blocks);
  return c;
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
  const QkCut c = cut_of(a, vec, vec ? 4 : 2, 3, 1 << 30);
  auto kern = a.f32 ? (vec ? qk_norm_fwd_kernel<float, true> : qk_norm_fwd_kernel<float, false>)
                    : (vec ? qk_norm_fwd_kernel<__nv_bfloat16, true> : qk_norm_fwd_kernel<__nv_bfloat16, false>);
  return launch_chained(kern, c.q_blocks + c.k_blocks, QKN_THREADS, 0, stream, a, c);
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
  const QkCut c = cut_of(a, vec, 2, 1, a.sum_rows);
  if (c.q_blocks + c.k_blocks > a.sum_rows) return -5;
  auto kern = a.f32 ? (vec ? qk_norm_bwd_ring_kernel<float> : qk_norm_bwd_kernel<float>)
                    : (vec ? qk_norm_bwd_ring_kernel<__nv_bfloat16> : qk_norm_bwd_kernel<__nv_bfloat16>);
  if (const int rc = launch_chained(kern, c.q_blocks + c.k_blocks, QKN_THREADS, 0, stream, a, c)) return rc;
  const bool shared = a.dwq == a.dwk;
  if (const int rc = launch_chained(qk_norm_sums_kernel, dim3((a.d + 31) / 32, shared ? 1 : 2), 1024, 0, stream, a.sums,
                                    c.q_blocks + (shared ? c.k_blocks : 0), c.k_blocks, a.d, a.dwq, a.dwk, a.add_dw))
    return rc;
  return 2;
}
