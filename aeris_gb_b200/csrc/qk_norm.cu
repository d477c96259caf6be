// RMS norms of queries and keys over each head's channels, with the position rotation in the same pass, and its gradients.
//
//   forward    z = w * x * r, r = (mean(x^2) + eps)^-1/2 over the head's d channels; y = R z, where R turns the channel pair
//              (2i, 2i + 1) by the angle of table row `pos` (i < rot / 2; channels from rot on are left as they are)
//   backward   dz = R^T dy; dw = sum over rows and heads of dz * x * r; with g = dz * w:
//              dx = r * (g - x r * mean(g x r))
//
// Both are bound by memory: 4 bytes of bf16 traffic an element forward, 6 backward, for about ten operations. A group of lanes
// (d / 8 of them, mostly rounded up to a power of two) owns one head of a row at a time, eight channels to a lane, so that a head
// is one or two loads a lane, its sum of squares a few shuffles, and a pair to be turned lies in one lane. A row's heads are cut
// into parts of q or of k alone, one of each where rows fill the GPU, down to one step each where they are few (single tokens); a block
// stays with its part and its warps walk over rows, so that a lane's weights, and in the backward pass its sums for dw, are one
// set of eight registers, strides are uniform, and angles are read once a row. Few heads leave a warp room for several rows a step
// (200,000 rows of 8 + 2 heads of 8: 93 us a row a step, 19 so). q and k have blocks in proportion to the time of a row. Everything
// between load and store is fp32. 64,800 rows of 24 + 24 heads of 64, bf16: forward 135 us, 5.9 TB/s (90 % of what a plain copy
// reaches); backward 214 us, 5.6 TB/s; 28,800 rows of 40 + 40 heads of 128 backward 319 us. fp32: 5.3 to 6 TB/s both ways from 64
// channels on. bf16 less where lanes or steps stay empty, 3.8 to 4.8 TB/s with heads of 72 to 104, 2 to 4 with heads of 16 to 36, and
// where a row has few heads, for a forward warp has the loads of one row under way (8 + 2 heads of 64: 4.1, stalls on loads first, 62 %
// of the issue slots taken, 41 % of DRAM); 0.4 to 1.4 where heads are not whole fours. One row, or one window of 900, takes the GPU 2 to
// 4 us, less than the host needs (12).
#include "api.h"
#include "common.cuh"
#include "host.h"

#include <type_traits>

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

// A lane's channels by what loads side by side, W: 8 (one or two 16-byte loads) channels 8 i .. 8 i + 7; 4 (8 or 16 bytes) channels
// 4 i .. 4 i + 3 and, `next` channels on, 4 (group + i) .. where there are as many, so that each load and store of a group is one
// piece; 0 (any even width, any alignment) the pairs lane, lane + 32, .. of the whole warp, from the head's start on.
struct Lane {
  int i, d, next;
  bool second;
};
__device__ __forceinline__ float bf16_lo(uint32_t x) { return __uint_as_float(x << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }
template <typename T, int W> struct HeadRaw;
template <> struct HeadRaw<__nv_bfloat16, 8> {
  uint4 a;
  __device__ void load(const __nv_bfloat16* p, bool mine, const Lane&) {
    a = make_uint4(0, 0, 0, 0);
    if (mine) a = *reinterpret_cast<const uint4*>(p);
  }
  __device__ Eight get() const {
    return {{f2_pack(bf16_lo(a.x), bf16_lo(a.y)), f2_pack(bf16_lo(a.z), bf16_lo(a.w))},
            {f2_pack(bf16_hi(a.x), bf16_hi(a.y)), f2_pack(bf16_hi(a.z), bf16_hi(a.w))}};
  }
  static __device__ void pack(const Eight& v, uint32_t (&w)[4]) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float e0, e1, o0, o1;
      f2_unpack(v.e[k], e0, e1);
      f2_unpack(v.o[k], o0, o1);
      w[2 * k] = pack_bf16x2(e0, o0);
      w[2 * k + 1] = pack_bf16x2(e1, o1);
    }
  }
  static __device__ void store(__nv_bfloat16* p, bool mine, const Lane&, const Eight& v) {
    uint32_t w[4];
    pack(v, w);
    if (mine) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <> struct HeadRaw<__nv_bfloat16, 4> {
  uint2 a, b;
  __device__ void load(const __nv_bfloat16* p, bool mine, const Lane& l) {
    a = b = make_uint2(0, 0);
    if (mine) a = *reinterpret_cast<const uint2*>(p);
    if (mine && l.second) b = *reinterpret_cast<const uint2*>(p + l.next);
  }
  __device__ Eight get() const {
    return {{f2_pack(bf16_lo(a.x), bf16_lo(a.y)), f2_pack(bf16_lo(b.x), bf16_lo(b.y))},
            {f2_pack(bf16_hi(a.x), bf16_hi(a.y)), f2_pack(bf16_hi(b.x), bf16_hi(b.y))}};
  }
  static __device__ void store(__nv_bfloat16* p, bool mine, const Lane& l, const Eight& v) {
    uint32_t w[4];
    HeadRaw<__nv_bfloat16, 8>::pack(v, w);
    if (mine) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    if (mine && l.second) *reinterpret_cast<uint2*>(p + l.next) = make_uint2(w[2], w[3]);
  }
};
template <int W> struct FloatRaw {
  float4 a, b;
  __device__ void load(const float* p, bool mine, const Lane& l) {
    a = b = make_float4(0.f, 0.f, 0.f, 0.f);
    if (mine) a = *reinterpret_cast<const float4*>(p);
    if (mine && (W == 8 || l.second)) b = *reinterpret_cast<const float4*>(p + (W == 8 ? 4 : l.next));
  }
  __device__ Eight get() const { return {{f2_pack(a.x, a.z), f2_pack(b.x, b.z)}, {f2_pack(a.y, a.w), f2_pack(b.y, b.w)}}; }
  static __device__ void store(float* p, bool mine, const Lane& l, const Eight& v) {
    float4 x, y;
    f2_unpack(v.e[0], x.x, x.z);
    f2_unpack(v.o[0], x.y, x.w);
    f2_unpack(v.e[1], y.x, y.z);
    f2_unpack(v.o[1], y.y, y.w);
    if (mine) *reinterpret_cast<float4*>(p) = x;
    if (mine && (W == 8 || l.second)) *reinterpret_cast<float4*>(p + (W == 8 ? 4 : l.next)) = y;
  }
};
template <> struct HeadRaw<float, 8> : FloatRaw<8> {};
template <> struct HeadRaw<float, 4> : FloatRaw<4> {};
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
template <typename T> struct HeadRaw<T, 0> {
  float f[8];
  __device__ void load(const T* p, bool mine, const Lane& l) {
    const int d = mine ? l.d : 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int e = 2 * (j * 32 + l.i);
      f[2 * j] = e < d ? to_float(p[e]) : 0.f;
      f[2 * j + 1] = e < d ? to_float(p[e + 1]) : 0.f;
    }
  }
  __device__ Eight get() const { return eight_of(f); }
  static __device__ void store(T* p, bool mine, const Lane& l, const Eight& x) {
    float v[8];
    singles(x, v);
    const int d = mine ? l.d : 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int e = 2 * (j * 32 + l.i);
      if (e < d) {
        from_float(v[2 * j], p + e);
        from_float(v[2 * j + 1], p + e + 1);
      }
    }
  }
};

// First channel of the lane's pair j.
template <int W> __device__ __forceinline__ int pair_channel(const Lane& l, int j) {
  return W == 8 ? 8 * l.i + 2 * j : W == 4 ? 4 * l.i + (j & 2 ? l.next : 0) + 2 * (j & 1) : 2 * (j * 32 + l.i);
}

template <int W> __device__ __forceinline__ Eight load_weight(const void* w, int bf16, const Lane& l) {
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int e = pair_channel<W>(l, j / 2) + (j & 1);
    v[j] = e >= l.d ? 0.f : bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(w)[e])
                               : reinterpret_cast<const float*>(w)[e];
  }
  return eight_of(v);
}

// Row of the table for `row`, or -1 where there is no such row or its position lies outside (recorded in the status word).
__device__ __forceinline__ int table_row(const AerisQkNorm& a, int row) {
  if (row >= a.rows) return -1;
  if (!a.rot) return 0;
  if (!a.pos) return row % a.L;
  const long long p = a.pos64 ? reinterpret_cast<const long long*>(a.pos)[row] : reinterpret_cast<const int*>(a.pos)[row];
  if (p >= 0 && p < a.L) return static_cast<int>(p);
  atomicCAS(a.status, 0, ERR_BOUNDS);
  return -1;
}

struct Angles {
  uint64_t c[2], s[2];                        // of pairs 0 and 1, of pairs 2 and 3
};
// Which of the lane's pairs are turned, a bit each.
template <int W> __device__ __forceinline__ int turned_pairs(const AerisQkNorm& a, const Lane& l) {
  int bits = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) bits |= (pair_channel<W>(l, j) < a.rot) << j;
  return bits;
}
// The pairs turned by their angles, back with BACK. A pair that is not turned has no part in it, not even times zero: an
// infinity or NaN in one of its channels is none in the other.
template <bool BACK> __device__ __forceinline__ void turn_pair(uint64_t& e, uint64_t& o, uint64_t c, uint64_t s, uint64_t mask) {
  const uint64_t x = f2_mul(o & mask, s), y = f2_mul(e & mask, s);
  e = f2_fma(e, c, BACK ? x : f2_neg(x));
  o = f2_fma(o, c, BACK ? f2_neg(y) : y);
}
// TURN: how much of a head is turned, 0 nothing, 1 a part, 2 all of it. A kernel of its own for each: the branch or the masks of the
// second cost it 6 % (24 + 24 heads of 64, 32 channels turned, bf16: forward 132 us without them, 140; by masks alone 140 too,
// backward 200, 209, 212), and asked for in heads that are turned as a whole they cost the backward pass as much.
template <int W, int TURN, bool BACK> __device__ __forceinline__ void turn(Eight& v, const Angles& r, int turned) {
  if (!TURN || (TURN == 1 && W == 8 && !turned)) return;              // by eights a lane turns all its pairs or none
#pragma unroll
  for (int k = 0; k < 2; ++k)
    turn_pair<BACK>(v.e[k], v.o[k], r.c[k], r.s[k],
                    TURN == 2 || W == 8 ? ~uint64_t(0)
                                        : (turned >> (2 * k) & 1 ? 0xffffffffull : 0) | (turned >> (2 * k) & 2 ? 0xffffffff00000000ull : 0));
}
template <int W, bool PAIRS> __device__ __forceinline__ Angles load_angles(const AerisQkNorm& a, int row, const Lane& l) {
  const long long at = row;
  float c[4], s[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    c[j] = 1.f;
    s[j] = 0.f;
  }
  if (W == 8) {                               // rot is a multiple of 8 here: a lane turns all its pairs or none
    if (8 * l.i < a.rot) {
      const float4 x = *reinterpret_cast<const float4*>(a.cos + at * (a.rot / 2) + 4 * l.i);
      const float4 y = *reinterpret_cast<const float4*>(a.sin + at * (a.rot / 2) + 4 * l.i);
      c[0] = x.x; c[1] = x.y; c[2] = x.z; c[3] = x.w;
      s[0] = y.x; s[1] = y.y; s[2] = y.z; s[3] = y.w;
    }
  } else if (W == 4 && PAIRS && a.rot % 4 == 0 && ((reinterpret_cast<uintptr_t>(a.cos) | reinterpret_cast<uintptr_t>(a.sin)) & 7) == 0) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int p = (4 * l.i + h * l.next) / 2;
      if (p < a.rot / 2) {
        const float2 x = *reinterpret_cast<const float2*>(a.cos + at * (a.rot / 2) + p);
        const float2 y = *reinterpret_cast<const float2*>(a.sin + at * (a.rot / 2) + p);
        c[2 * h] = x.x; c[2 * h + 1] = x.y;
        s[2 * h] = y.x; s[2 * h + 1] = y.y;
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int p = pair_channel<W>(l, j) / 2;
      if (p < a.rot / 2) {
        c[j] = a.cos[at * (a.rot / 2) + p];
        s[j] = a.sin[at * (a.rot / 2) + p];
      }
    }
  }
  return {{f2_pack(c[0], c[1]), f2_pack(c[2], c[3])}, {f2_pack(s[0], s[1]), f2_pack(s[2], s[3])}};
}

// What a block works on: `steps` steps of `per_step` heads of q or k, from head `first` on; its warps take rows `row`, row +
// stride, .. Where a row has half as many heads as a step takes or fewer, a step takes heads of `q_rows` or `k_rows` rows instead,
// and `row` is a lane's own: the rows of a warp begin at row - row_sub.
struct QkCut {
  int group, per_step;                                  // lanes a head, heads a step
  int q_len, k_len, q_blocks, k_blocks, q_rows, k_rows;      // steps of a part, blocks of all parts, rows a step of q and of k
};
struct Part {
  Lane lane;
  int head, first, steps, heads, row, row_sub, stride;       // heads: what is left from the lane's first one on, 0: none
  bool is_k;
  template <int W> static __device__ Part make(const AerisQkNorm& a, const QkCut& cut) {
    Part t;
    const int lane = threadIdx.x & 31, slot = lane / cut.group, i = lane - slot * cut.group;
    t.lane = {i, a.d, 4 * cut.group, 4 * (cut.group + i) < a.d};
    t.is_k = blockIdx.x >= cut.q_blocks;
    const int heads = t.is_k ? a.kv_heads : a.heads, at_once = t.is_k ? cut.k_rows : cut.q_rows;
    const int len = t.is_k ? cut.k_len : cut.q_len, all = (heads + cut.per_step - 1) / cut.per_step, parts = (all + len - 1) / len;
    const int block = t.is_k ? blockIdx.x - cut.q_blocks : blockIdx.x;
    const int step = block % parts * len;
    t.steps = min(len, all - step);
    t.first = step * cut.per_step;
    t.row_sub = at_once > 1 ? min(slot / heads, at_once - 1) : 0;
    t.head = slot - t.row_sub * (at_once > 1 ? heads : 0);
    t.heads = slot >= cut.per_step || (W == 8 && 8 * i >= a.d) ? 0 : max(0, heads - t.first - t.head);
    t.row = (block / parts * QKN_WARPS + (threadIdx.x >> 5)) * at_once + t.row_sub;
    t.stride = (t.is_k ? cut.k_blocks : cut.q_blocks) / parts * QKN_WARPS * at_once;   // the blocks are a multiple of the parts
    return t;
  }
};
template <typename T, int W> __device__ __forceinline__ T* lane_start(const AerisHeads& t, const Part& w) {
  return reinterpret_cast<T*>(const_cast<void*>(t.ptr)) + w.row * t.row + (w.first + w.head) * t.head + W * w.lane.i;
}

// Sums over a head's lanes, in each of them; ODD: they may be no power of two.
template <bool ODD, int N> __device__ __forceinline__ void group_sums(float (&v)[N], int i, const QkCut& cut) {
  if (!ODD) {
    for (int o = cut.group >> 1; o > 0; o >>= 1)
#pragma unroll
      for (int k = 0; k < N; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
    return;
  }
  const int lane = threadIdx.x & 31;
  for (int n = cut.group; n > 1;) {
    const int half = (n + 1) >> 1;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const float other = __shfl_sync(0xffffffffu, v[k], lane + half);
      if (i + half < n) v[k] += other;
    }
    n = half;
  }
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = __shfl_sync(0xffffffffu, v[k], lane - i);
}

// Blocks an SM of the forward kernel; fp32 by fours needs more registers for the heads in flight.
template <typename T, int W> constexpr int fwd_blocks() { return W == 0 ? 2 : W == 4 && sizeof(T) == 4 ? 3 : 4; }

template <typename T, int W, bool ODD, int TURN>
__global__ void __launch_bounds__(QKN_THREADS, fwd_blocks<T, W>()) qk_norm_fwd_kernel(const AerisQkNorm a, const QkCut cut) {
  constexpr int U = W ? 3 : 2;                // heads in flight per lane
  const Part t = Part::make<W>(a, cut);
  const AerisHeads in = t.is_k ? a.k : a.q, out = t.is_k ? a.k_out : a.q_out;
  const T* x_row = lane_start<const T, W>(in, t);
  T* y_row = lane_start<T, W>(out, t);
  const float inv_d = 1.f / a.d;
  chain_point();
  const Eight w = load_weight<W>(t.is_k ? a.wk : a.wq, a.w_bf16, t.lane);
  const int turned = TURN == 1 ? turned_pairs<W>(a, t.lane) : 0;
  for (int row = t.row; row - t.row_sub < a.rows; row += t.stride, x_row += t.stride * in.row, y_row += t.stride * out.row) {
    const int at = table_row(a, row);         // nothing but the angles waits for it
    const int heads = row < a.rows ? t.heads : 0;
    const Angles r = load_angles<W, sizeof(T) == 2>(a, max(at, 0), t.lane);
    const T* x = x_row;
    T* y = y_row;
#pragma unroll 1
    for (int step = 0; step < t.steps; step += U) {
      HeadRaw<T, W> raw[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        raw[u].load(x + u * (cut.per_step * in.head), step + u < t.steps && (step + u) * cut.per_step < heads, t.lane);
      x += U * (cut.per_step * in.head);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (step + u >= t.steps) break;
        Eight v = raw[u].get();
        const uint64_t ss = f2_fma(v.o[1], v.o[1], f2_fma(v.e[1], v.e[1], f2_fma(v.o[0], v.o[0], f2_mul(v.e[0], v.e[0]))));
        float sum[1] = {f2_sum(ss)};
        group_sums<ODD>(sum, t.lane.i, cut);
        const uint64_t scale = f2_all(rsqrtf(sum[0] * inv_d + a.eps));
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          v.e[k] = f2_mul(f2_mul(v.e[k], scale), w.e[k]);
          v.o[k] = f2_mul(f2_mul(v.o[k], scale), w.o[k]);
        }
        turn<W, TURN, false>(v, r, turned);
        HeadRaw<T, W>::store(y + u * (cut.per_step * out.head), at >= 0 && (step + u) * cut.per_step < heads, t.lane, v);
      }
      y += U * (cut.per_step * out.head);
    }
  }
}

// One head's gradient in a lane: v = x and g = dy on entry; dw is added to, g holds dx on return. Not `live`: a place without a
// head, all zeros, whose root without eps would be infinite.
template <int W, bool ODD, int TURN>
__device__ __forceinline__ void head_backward(const Eight& v, Eight& g, const Eight& w, const Angles& r, int turned, Eight& dw, int i,
                                              const QkCut& cut, bool live, float inv_d, float eps) {
  uint64_t ss2 = 0, dot2 = 0;                 // two zeros
  Eight gw;
  turn<W, TURN, true>(g, r, turned);
  // mean(g x r) needs no r before its sum: both sums go through the shuffles together
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    gw.e[k] = f2_mul(g.e[k], w.e[k]);
    gw.o[k] = f2_mul(g.o[k], w.o[k]);
    ss2 = f2_fma(v.o[k], v.o[k], f2_fma(v.e[k], v.e[k], ss2));
    dot2 = f2_fma(gw.o[k], v.o[k], f2_fma(gw.e[k], v.e[k], dot2));
  }
  float sum[2] = {f2_sum(ss2), f2_sum(dot2)};
  group_sums<ODD>(sum, i, cut);
  const float scale = live ? rsqrtf(sum[0] * inv_d + eps) : 0.f;
  const uint64_t s2 = f2_all(scale), m2 = f2_all(-sum[1] * inv_d * scale * scale);
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
template <int W>
__device__ __forceinline__ void block_sums(float (*red)[QKN_MAX_D], const Eight& sum8, const Lane& l, const QkCut& cut, float* sums) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d = l.d;
  float dw[8];
  singles(sum8, dw);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    float sum = dw[j];
    for (int k = 1; k < cut.per_step; ++k) sum += __shfl_sync(0xffffffffu, dw[j], lane + k * cut.group);
    const int e = pair_channel<W>(l, j / 2) + (j & 1);
    if (lane < cut.group && e < d) red[warp][e] = sum;
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
template <typename T, int TURN>
__global__ void __launch_bounds__(QKN_THREADS, 2) qk_norm_bwd_kernel(const AerisQkNorm a, const QkCut cut) {
  __shared__ float red[QKN_WARPS][QKN_MAX_D];
  const Part t = Part::make<0>(a, cut);
  const AerisHeads in = t.is_k ? a.k : a.q, grad = t.is_k ? a.dk : a.dq, out = t.is_k ? a.k_out : a.q_out;
  const T *x = lane_start<const T, 0>(in, t), *dy = lane_start<const T, 0>(grad, t);
  T* dx = lane_start<T, 0>(out, t);
  const float inv_d = 1.f / a.d;
  chain_point();
  const Eight w = load_weight<0>(t.is_k ? a.wk : a.wq, a.w_bf16, t.lane);
  const int turned = TURN == 1 ? turned_pairs<0>(a, t.lane) : 0;
  Eight dw = {};
  for (int row = t.row; row < a.rows; row += t.stride, x += t.stride * in.row, dy += t.stride * grad.row, dx += t.stride * out.row) {
    const int at = table_row(a, row);
    if (at < 0) continue;
    const Angles r = load_angles<0, false>(a, at, t.lane);
#pragma unroll 1
    for (int step = 0; step < t.steps; ++step) {        // a head a step here
      HeadRaw<T, 0> rx, rg;
      rx.load(x + step * in.head, true, t.lane);
      rg.load(dy + step * grad.head, true, t.lane);
      Eight g = rg.get();
      head_backward<0, false, TURN>(rx.get(), g, w, r, turned, dw, t.lane.i, cut, true, inv_d, a.eps);
      HeadRaw<T, 0>::store(dx + step * out.head, true, t.lane, g);
    }
  }
  block_sums<0>(red, dw, t.lane, cut, a.sums);
}

// Whole vectors. What a warp reads passes through a ring of its own in shared memory, a few steps ahead (asynchronous copies
// of 16 bytes that the same lane takes out again): with the loads in registers, two steps at a time, 127 registers left 16
// warps per SM too little under way (64,800 rows, 24 + 24 heads of 64: 265 us; ring 247, with two-wide arithmetic 212 to 217;
// three blocks an SM instead of two 217 where that took 212).
template <typename T, int W, bool ODD, int TURN>
__global__ void __launch_bounds__(QKN_THREADS, 2) qk_norm_bwd_ring_kernel(const AerisQkNorm a, const QkCut cut) {
  constexpr int VECS = W == 8 ? 1 : 2, BYTES = W * sizeof(T);         // copies a head and lane, and their size
  constexpr int AHEAD = VECS * BYTES == 16 ? 4 : 3;                   // stages of the ring
  __shared__ union {
    uint4 ring[QKN_WARPS][AHEAD][2][VECS][2 * BYTES];                 // 32 lanes' of BYTES each
    float red[QKN_WARPS][QKN_MAX_D];
  } sm;
  const Part t = Part::make<W>(a, cut);
  const AerisHeads in = t.is_k ? a.k : a.q, grad = t.is_k ? a.dk : a.dq, out = t.is_k ? a.k_out : a.q_out;
  const T *x = lane_start<const T, W>(in, t), *dy = lane_start<const T, W>(grad, t);      // of the copies ahead
  T* dx = lane_start<T, W>(out, t);
  const float inv_d = 1.f / a.d;
  uint4 (*ring)[2][VECS][2 * BYTES] = sm.ring[threadIdx.x >> 5];
  chain_point();
  const Eight w = load_weight<W>(t.is_k ? a.wk : a.wq, a.w_bf16, t.lane);
  const int turned = TURN == 1 ? turned_pairs<W>(a, t.lane) : 0;
  Eight dw = {};
  const long long in_step = cut.per_step * in.head, grad_step = cut.per_step * grad.head, out_step = cut.per_step * out.head;
  int ahead_row = t.row, ahead_step = 0;
  uint32_t ahead_to = smem_u32(ring) + (threadIdx.x & 31) * BYTES;
  const uint32_t ring_end = ahead_to + AHEAD * sizeof(ring[0]);
  uint32_t from = ahead_to;
  auto next = [&](uint32_t slot) { return slot + sizeof(ring[0]) == ring_end ? ring_end - AHEAD * sizeof(ring[0]) : slot + sizeof(ring[0]); };
  auto take = [](uint32_t to, const T* p) {
    if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(p) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(to), "l"(p) : "memory");
  };
  auto copy = [&] {
    if (ahead_row - t.row_sub < a.rows) {
      if (ahead_step * cut.per_step < t.heads && ahead_row < a.rows) {
        take(ahead_to, x);
        take(ahead_to + 32 * VECS * BYTES, dy);
        if (VECS == 2 && t.lane.second) {
          take(ahead_to + 32 * BYTES, x + t.lane.next);
          take(ahead_to + 96 * BYTES, dy + t.lane.next);
        }
      }
      x += in_step;
      dy += grad_step;
      if (++ahead_step == t.steps) {
        ahead_step = 0;
        ahead_row += t.stride;
        x += t.stride * in.row - t.steps * in_step;
        dy += t.stride * grad.row - t.steps * grad_step;
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    ahead_to = next(ahead_to);
  };
#pragma unroll
  for (int k = 0; k < AHEAD - 1; ++k) copy();
  const Lane in_ring = {t.lane.i, a.d, 32 * W, t.lane.second};
  int next_at = table_row(a, t.row);
  for (int row = t.row; row - t.row_sub < a.rows; row += t.stride, dx += t.stride * out.row - t.steps * out_step) {
    const int at = next_at, heads = at < 0 ? 0 : t.heads;
    next_at = table_row(a, row + t.stride);
    const Angles r = load_angles<W, sizeof(T) == 2>(a, max(at, 0), t.lane);
#pragma unroll 1
    for (int step = 0; step < t.steps; ++step, dx += out_step) {
      copy();
      asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD - 1) : "memory");
      const bool mine = step * cut.per_step < heads;
      const T* slot = reinterpret_cast<const T*>(__cvta_shared_to_generic(from));
      HeadRaw<T, W> rx, rg;
      rx.load(slot, mine, in_ring);
      rg.load(slot + 32 * VECS * W, mine, in_ring);
      Eight g = rg.get();
      // lanes behind the head's width hold zeros and have their head's root
      head_backward<W, ODD, TURN>(rx.get(), g, w, r, turned, dw, t.lane.i, cut, mine, inv_d, a.eps);
      HeadRaw<T, W>::store(dx, mine, t.lane, g);
      from = next(from);
    }
  }
  __syncthreads();                            // the ring becomes the sums' place
  block_sums<W>(sm.red, dw, t.lane, cut, a.sums);
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

bool whole(const AerisHeads& t, int size, int bytes) {
  return reinterpret_cast<uintptr_t>(t.ptr) % bytes == 0 && (t.row * size) % bytes == 0 && (t.head * size) % bytes == 0;
}
bool angles_in_vectors(const AerisQkNorm& a) {
  return !a.rot || (a.rot % 8 == 0 && reinterpret_cast<uintptr_t>(a.cos) % 16 == 0 && reinterpret_cast<uintptr_t>(a.sin) % 16 == 0);
}
// Channels that load side by side, see Lane. fp32 backward goes by four: a group's two loads are a piece each then, where halves of
// 32 bytes come twice through L2 (copies pass L1 by; 65,000 rows of 12 + 12 heads of 64 by eight 307 us, by four 210). Forward
// L1 has the second half, and by eight is the faster (12,345 rows of 10 + 2 heads of 72, 40 channels turned: 23.5 us, by four 27.8).
int width_of(const AerisQkNorm& a, bool grad) {
  const int size = a.f32 ? 4 : 2;
  auto all = [&](int w) {
    const int bytes = w * size < 16 ? w * size : 16;
    return a.d % w == 0 && whole(a.q, size, bytes) && whole(a.k, size, bytes) && whole(a.q_out, size, bytes) &&
           whole(a.k_out, size, bytes) && (!grad || (whole(a.dq, size, bytes) && whole(a.dk, size, bytes)));
  };
  return !(a.f32 && grad) && angles_in_vectors(a) && all(8) ? 8 : all(4) ? 4 : 0;
}

// Widths of which half as many heads again fit a step when their lanes are not rounded up to a power of two: five lanes (40
// channels), nine and ten (72 and 80). There it pays for the longer way to a sum (12 + 12 heads of 72, bf16, rounded up / not: forward
// 212 / 192 us, backward 352 / 294), with a quarter more it does not (heads of 48, five a step for four: 274 / 324).
bool odd(int d) {
  const int lanes = (d + 7) / 8;
  int group = 1;
  while (group < lanes) group *= 2;
  return 2 * (32 / lanes) >= 3 * (32 / group);
}

// Lanes per head, parts and blocks: `most` blocks in all, or the few that one row a warp and one step a part make. A row takes a
// warp as long as its steps and `own` more for the row itself, which the shares of q and k go by: with heads alone, two key heads
// next to eight of queries got a fifth of the blocks, and took longer than those (156,250 rows of 8 + 2 heads of 128, backward: 296
// us by heads, 244 with one step more; forward 193 with one, 171 with two).
QkCut cut_of(const AerisQkNorm& a, int width, int blocks_per_sm, double own, int most) {
  QkCut c;
  c.group = 32;
  if (width) {
    const int lanes = (a.d + 7) / 8;
    for (c.group = 1; c.group < lanes;) c.group *= 2;
    if (odd(a.d)) c.group = lanes;
  }
  c.per_step = 32 / c.group;
  const int per = c.per_step, q = (a.heads + per - 1) / per, k = (a.kv_heads + per - 1) / per;
  c.q_rows = per / a.heads > 1 ? per / a.heads : 1;
  c.k_rows = per / a.kv_heads > 1 ? per / a.kv_heads : 1;
  int cap = num_sms() * blocks_per_sm;
  if (cap > most) cap = most;
  auto side = [&](int steps, int rows, int share, int& len, int& blocks) {
    if (share < 1) share = 1;
    const long long row_blocks = (a.rows + QKN_WARPS * rows - 1) / (QKN_WARPS * rows);
    const long long want = (share + row_blocks - 1) / row_blocks;               // parts that fill the share
    const int parts = static_cast<int>(want < steps ? want : steps);
    len = (steps + parts - 1) / parts;
    const int real = (steps + len - 1) / len;
    const long long by_rows = share / real < 1 ? 1 : share / real;
    blocks = real * static_cast<int>(row_blocks < by_rows ? row_blocks : by_rows);
  };
  const double q_time = (own + q) / c.q_rows, k_time = (own + k) / c.k_rows;
  const int q_share = static_cast<int>(cap * (q_time / (q_time + k_time)));
  side(q, c.q_rows, q_share, c.q_len, c.q_blocks);
  side(k, c.k_rows, cap - q_share, c.k_len, c.k_blocks);
  return c;
}

template <int N> using Int = std::integral_constant<int, N>;
template <typename F> auto by_turn(const AerisQkNorm& a, F f) {
  return !a.rot ? f(Int<0>{}) : a.rot < a.d ? f(Int<1>{}) : f(Int<2>{});
}

int refused(const AerisQkNorm& a) {
  if (a.rows <= 0 || a.rows > 0x7fffffff - (1 << 20) || a.heads <= 0 || a.kv_heads <= 0 || a.d <= 0 || a.d % 2 || a.d > QKN_MAX_D) return -1;
  if (a.rot < 0 || a.rot % 2 || a.rot > a.d || (a.rot && (!a.cos || !a.sin || a.L <= 0)) || !a.wq || !a.wk) return -2;
  if (!a.q.ptr || !a.k.ptr || !a.q_out.ptr || !a.k_out.ptr || !a.status) return -3;
  return 0;
}

}  // namespace
}  // namespace aeris

using namespace aeris;

extern "C" int aeris_qk_norm_fwd(const AerisQkNorm* p, void* stream_) {
  const AerisQkNorm& a = *p;
  if (const int rc = refused(a)) return rc;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  const int w = width_of(a, false);
  const QkCut c = cut_of(a, w, !w ? 2 : a.f32 && w == 4 ? 3 : 4, 2, 1 << 30);
  using bf16 = __nv_bfloat16;
  auto pick = [&](auto t, auto width, auto turn) {
    constexpr int W = decltype(width)::value, TURN = decltype(turn)::value;
    using T = decltype(t);
    return W && odd(a.d) ? qk_norm_fwd_kernel<T, W, W != 0, TURN> : qk_norm_fwd_kernel<T, W, false, TURN>;
  };
  auto by_width = [&](auto t, auto turn) {
    return w == 8 ? pick(t, Int<8>{}, turn) : w ? pick(t, Int<4>{}, turn) : pick(t, Int<0>{}, turn);
  };
  auto by_type = [&](auto turn) { return a.f32 ? by_width(0.f, turn) : by_width(bf16(), turn); };
  // Heads by eights of which nothing is turned go through the kernel with the branch: 65,000 rows of 24 + 24 heads of 64 take 127 us
  // there and 146 without it, where all of a step's stores come at once.
  auto kern = w == 8 && !a.rot ? by_type(Int<1>{}) : by_turn(a, by_type);
  return launch_chained(kern, c.q_blocks + c.k_blocks, QKN_THREADS, 0, stream, a, c);
}

// Returns the number of kernels launched, or a negative code.
extern "C" int aeris_qk_norm_bwd(const AerisQkNorm* p, void* stream_) {
  const AerisQkNorm& a = *p;
  if (const int rc = refused(a)) return rc;
  if (!a.dq.ptr || !a.dk.ptr || !a.dwq || !a.dwk || !a.sums || a.sum_rows <= 0) return -4;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  const int w = width_of(a, true);
  const QkCut c = cut_of(a, w, 2, 1, a.sum_rows);
  if (c.q_blocks + c.k_blocks > a.sum_rows) return -5;
  using bf16 = __nv_bfloat16;
  auto ring = [&](auto t, auto width, auto turn) {
    constexpr int W = decltype(width)::value, TURN = decltype(turn)::value;
    using T = decltype(t);
    return odd(a.d) ? qk_norm_bwd_ring_kernel<T, W, true, TURN> : qk_norm_bwd_ring_kernel<T, W, false, TURN>;
  };
  auto kern = by_turn(a, [&](auto turn) {
    constexpr int TURN = decltype(turn)::value;
    return a.f32 ? (w ? ring(0.f, Int<4>{}, turn) : qk_norm_bwd_kernel<float, TURN>)
                 : (w == 8 ? ring(bf16(), Int<8>{}, turn) : w ? ring(bf16(), Int<4>{}, turn) : qk_norm_bwd_kernel<bf16, TURN>);
  });
  if (const int rc = launch_chained(kern, c.q_blocks + c.k_blocks, QKN_THREADS, 0, stream, a, c)) return rc;
  const bool shared = a.dwq == a.dwk;
  if (const int rc = launch_chained(qk_norm_sums_kernel, dim3((a.d + 31) / 32, shared ? 1 : 2), 1024, 0, stream, a.sums,
                                    c.q_blocks + (shared ? c.k_blocks : 0), c.k_blocks, a.d, a.dwq, a.dwk, a.add_dw))
    return rc;
  return 2;
}
