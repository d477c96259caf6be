// Layer norm of rows that lie in registers. Included by layer_norm.cu.
//
// Memory is the floor: a row is read once (forward) or with its gradient once (backward) and written once. Rows are taken in
// vectors of 16 bytes where they start on 16-byte boundaries and consist of whole ones, else element by element; a lane has up to
// NV of them. Narrow rows share a warp (a group of lanes each), rows up to 32 NV vectors take a warp, wider ones a block of up to 1,024 threads.
#pragma once

namespace aeris {

namespace {

// One vector of a row: W elements, as pairs of fp32.
template <typename T> struct RowVec;
template <> struct RowVec<__nv_bfloat16> {
  uint4 r;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { r = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void get(uint64_t (&f)[4]) const {
    f[0] = f2_from_bf16x2(r.x); f[1] = f2_from_bf16x2(r.y); f[2] = f2_from_bf16x2(r.z); f[3] = f2_from_bf16x2(r.w);
  }
  static __device__ __forceinline__ void store(__nv_bfloat16* p, const uint64_t (&f)[4]) {
    *reinterpret_cast<uint4*>(p) = make_uint4(f2_to_bf16x2(f[0]), f2_to_bf16x2(f[1]), f2_to_bf16x2(f[2]), f2_to_bf16x2(f[3]));
  }
};
template <> struct RowVec<float> {
  ulonglong2 r;
  __device__ __forceinline__ void load(const float* p) { r = *reinterpret_cast<const ulonglong2*>(p); }
  __device__ __forceinline__ void get(uint64_t (&f)[2]) const { f[0] = r.x; f[1] = r.y; }
  static __device__ __forceinline__ void store(float* p, const uint64_t (&f)[2]) {
    *reinterpret_cast<ulonglong2*>(p) = make_ulonglong2(f[0], f[1]);
  }
};

// W elements of the weight or the bias from column c on.
template <int W>
__device__ __forceinline__ void load_weights(const void* w, int f32, int c, uint64_t (&f)[W / 2]) {
  if (f32) {
    const ulonglong2* p = reinterpret_cast<const ulonglong2*>(static_cast<const float*>(w) + c);
#pragma unroll
    for (int i = 0; i < W / 4; ++i) {
      const ulonglong2 v = p[i];
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    }
  } else if constexpr (W == 8) {
    const uint4 v = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(w) + c);
    f[0] = f2_from_bf16x2(v.x); f[1] = f2_from_bf16x2(v.y); f[2] = f2_from_bf16x2(v.z); f[3] = f2_from_bf16x2(v.w);
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(w) + c);
    f[0] = f2_from_bf16x2(v.x); f[1] = f2_from_bf16x2(v.y);
  }
}
__device__ __forceinline__ float f2_sum(uint64_t v) {
  float a, b;
  f2_unpack(v, a, b);
  return a + b;
}
__device__ __forceinline__ uint64_t f2_both(float v) { return f2_pack(v, v); }

struct LnCut {
  int group;        // lanes of a row (a power of two up to 32), or 0: the block
  int rows;         // rows of a block at a time
};

// Sum over the lanes of a row, in each of them. `part`: 32 words for every value that is summed at once (block only).
template <bool BLOCK, int K>
__device__ __forceinline__ void row_sums(float (&v)[K], int group, float* part) {
  if constexpr (!BLOCK) {
    for (int o = group >> 1; o > 0; o >>= 1)
#pragma unroll
      for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  } else {
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = warp_sum(v[k]);
    __syncthreads();        // the words may still be read from the sum before
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int k = 0; k < K; ++k) part[k * 32 + (threadIdx.x >> 5)] = v[k];
    __syncthreads();
    const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = warp_sum(lane < warps ? part[k * 32 + lane] : 0.f);
  }
}

// A row per group of lanes (BLOCK = false: 8 warps) or per block. Lane l has vectors l, l + lanes, .. Issue slots bound it beside
// memory (62 % of them, 64,800 rows of 1536, bf16: 80 us, 5.0 TB/s): arithmetic is two-wide, the differences from the mean take the
// row's place, and rows are whole vectors (with the differences taken twice and a last vector that may be cut off, whose
// predicated code is issued for all of them, 89 us). Tried: rows through a ring of bulk copies 140, a block per row 133,
// four blocks an SM (64 registers, spilled) 103.
template <typename T, int W, int NV, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? 1024 : 256) ln_fwd_kernel(const AerisLayerNorm a, const LnCut cut) {
  __shared__ float part[BLOCK ? 32 : 1];
  constexpr int P = W / 2;
  chain_point();
  const int lanes = BLOCK ? blockDim.x : cut.group, lane = BLOCK ? threadIdx.x : threadIdx.x & (cut.group - 1);
  const long long row = BLOCK ? blockIdx.x : static_cast<long long>(blockIdx.x) * cut.rows + threadIdx.x / cut.group;
  const bool live = row < a.rows;       // lanes of rows that there are not stay for the sums of their warp
  const T* x = static_cast<const T*>(a.x) + (live ? row : 0) * a.ld_x;
  uint64_t v[NV][P];
  {
    RowVec<T> raw[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * lanes + lane) * W;
      if (c < a.cols) raw[i].load(x + c);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if ((i * lanes + lane) * W < a.cols) {
        raw[i].get(v[i]);
      } else {
#pragma unroll
        for (int k = 0; k < P; ++k) v[i][k] = 0ull;
      }
    }
  }
  constexpr bool EARLY = BLOCK && NV == 1;        // weight and bias are asked for with the row
  uint64_t we[P], be[P];
  if constexpr (EARLY) {
    const int c = lane * W;
    if (a.w && c < a.cols) load_weights<W>(a.w, a.w_f32, c, we);
    if (a.b && c < a.cols) load_weights<W>(a.b, a.w_f32, c, be);
  }
  const float inv = 1.f / static_cast<float>(a.cols);
  uint64_t t = 0ull;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int k = 0; k < P; ++k) t = f2_add(t, v[i][k]);
  float s[1] = {f2_sum(t)};
  row_sums<BLOCK, 1>(s, cut.group, part);
  const float mean = s[0] * inv;
  const uint64_t m = f2_both(mean);
  t = 0ull;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if ((i * lanes + lane) * W < a.cols) {
#pragma unroll
      for (int k = 0; k < P; ++k) {
        v[i][k] = f2_sub(v[i][k], m);
        t = f2_fma(v[i][k], v[i][k], t);
      }
    }
  }
  s[0] = f2_sum(t);
  row_sums<BLOCK, 1>(s, cut.group, part);
  const float rstd = 1.f / sqrtf(s[0] * inv + a.eps);
  if (!live) return;
  const uint64_t r = f2_both(rstd);
  T* y = static_cast<T*>(a.y) + row * a.ld_y;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * lanes + lane) * W;
    if (c < a.cols) {
      uint64_t w[P];
#pragma unroll
      for (int k = 0; k < P; ++k) v[i][k] = f2_mul(v[i][k], r);
      if (a.w) {
        if constexpr (!EARLY) load_weights<W>(a.w, a.w_f32, c, w);
#pragma unroll
        for (int k = 0; k < P; ++k) v[i][k] = f2_mul(v[i][k], EARLY ? we[k] : w[k]);
      }
      if (a.b) {
        if constexpr (!EARLY) load_weights<W>(a.b, a.w_f32, c, w);
#pragma unroll
        for (int k = 0; k < P; ++k) v[i][k] = f2_add(v[i][k], EARLY ? be[k] : w[k]);
      }
      RowVec<T>::store(y + c, v[i]);
    }
  }
  if (lane == 0) *reinterpret_cast<float2*>(a.stats + 2 * row) = make_float2(mean, rstd);
}

// The same element by element, for rows that start anywhere.
template <typename T, int NV, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? 1024 : 256) ln_fwd_one_kernel(const AerisLayerNorm a, const LnCut cut) {
  __shared__ float part[BLOCK ? 32 : 1];
  chain_point();
  const int lanes = BLOCK ? blockDim.x : cut.group, lane = BLOCK ? threadIdx.x : threadIdx.x & (cut.group - 1);
  const long long row = BLOCK ? blockIdx.x : static_cast<long long>(blockIdx.x) * cut.rows + threadIdx.x / cut.group;
  const bool live = row < a.rows;
  const T* x = static_cast<const T*>(a.x) + (live ? row : 0) * a.ld_x;
  float v[NV], s[1] = {0.f};
#pragma unroll
  for (int i = 0; i < NV; ++i) v[i] = i * lanes + lane < a.cols ? ld_f(x + i * lanes + lane) : 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) s[0] += v[i];
  const float inv = 1.f / static_cast<float>(a.cols);
  row_sums<BLOCK, 1>(s, cut.group, part);
  const float mean = s[0] * inv;
  s[0] = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (i * lanes + lane < a.cols) {
      v[i] -= mean;
      s[0] = fmaf(v[i], v[i], s[0]);
    }
  row_sums<BLOCK, 1>(s, cut.group, part);
  const float rstd = 1.f / sqrtf(s[0] * inv + a.eps);
  if (!live) return;
  T* y = static_cast<T*>(a.y) + row * a.ld_y;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = i * lanes + lane;
    if (c < a.cols) {
      float f = v[i] * rstd;
      if (a.w) f *= weight_at(a.w, a.w_f32, c);
      if (a.b) f += weight_at(a.b, a.w_f32, c);
      st_f(y + c, f);
    }
  }
  if (lane == 0) *reinterpret_cast<float2*>(a.stats + 2 * row) = make_float2(mean, rstd);
}

// The column sums of the only block.
__device__ __forceinline__ void column_sums(const AerisLayerNorm& a, int c, float dw, float db) {
  if (a.dw) a.dw[c] = a.add ? a.dw[c] + dw : dw;
  if (a.db) a.db[c] = a.add ? a.db[c] + db : db;
}

// Where the whole grid is one cluster, its CTAs' sums ([2, cols] in the shared memory of each) are added in their order; each has a
// part of the columns.
__device__ __forceinline__ void cluster_sums(const AerisLayerNorm& a, const float* joined) {
  __syncthreads();
  cluster_sync_all();
  const uint32_t mine = smem_u32(joined);
  for (int c = blockIdx.x * blockDim.x + threadIdx.x; c < a.cols; c += gridDim.x * blockDim.x) {
    float dw = 0.f, db = 0.f;
    for (uint32_t k = 0; k < gridDim.x; ++k) {
      const uint32_t at = map_to_cta(mine + c * 4, k);
      dw += ld_shared_cluster_f32(at);
      db += ld_shared_cluster_f32(at + a.cols * 4);
    }
    column_sums(a, c, dw, db);
  }
  cluster_sync_all();       // nobody leaves before the others have read
}

// The warps' column sums (of each warp's first group, which has those of the others), one after the other so that the order of
// additions is fixed, and the block's slice of `work`.
template <bool FEW, typename F>
__device__ __forceinline__ void join_warps(const AerisLayerNorm& a, float* joined, int lanes, F&& each) {
  const int warp = threadIdx.x >> 5;
  const bool first = static_cast<int>(threadIdx.x & 31) < lanes;
  for (int t = 0; t < static_cast<int>(blockDim.x >> 5); ++t) {
    if (warp == t && first)
      each([&](int c, float dw, float db) {
        joined[c] = t ? joined[c] + dw : dw;
        joined[a.cols + c] = t ? joined[a.cols + c] + db : db;
      });
    __syncthreads();
  }
  if constexpr (FEW) return cluster_sums(a, joined);
  float* out = a.work + static_cast<long long>(blockIdx.x) * 2 * a.cols;
  for (int c = threadIdx.x; c < 2 * a.cols; c += blockDim.x) out[c] = joined[c];
}

// Gradients. A thread keeps its columns for all rows that it sees (NV vectors), and their sums of dy xhat and dy in registers; R
// rows are taken at a time, so that their loads and the latencies of their sums are shared. MIN: blocks that an SM is to hold.
// FEW: the grid is a cluster that joins its sums, in code of its own (as a branch it cost many rows 133 -> 163 us).
// 64,800 rows of 1536, bf16: 132 us, 4.5 TB/s, and 5 for the slices' join; with two blocks an SM 153; the next rows asked for
// a round ahead 135 (R = 2); a warp per row and its sums in 170 registers 360.
template <typename T, int W, int NV, int R, bool BLOCK, int THREADS, int MIN, bool FEW>
__global__ void __launch_bounds__(THREADS, MIN) ln_bwd_kernel(const AerisLayerNorm a, const LnCut cut) {
  __shared__ float part[BLOCK ? 64 * R : 1];
  extern __shared__ float joined[];         // [2, cols] of a cluster's CTA, and where BLOCK = false
  constexpr int P = W / 2;
  constexpr bool KEEP = NV == 1;            // the weight stays in registers
  chain_point();
  const int lanes = BLOCK ? blockDim.x : cut.group, lane = BLOCK ? threadIdx.x : threadIdx.x & (cut.group - 1);
  const int group = BLOCK ? 0 : threadIdx.x / cut.group, groups = BLOCK ? 1 : cut.rows;
  const float inv = 1.f / static_cast<float>(a.cols);
  uint64_t dw[NV][P], db[NV][P], w[P];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int k = 0; k < P; ++k) dw[i][k] = db[i][k] = 0ull;
#pragma unroll
  for (int k = 0; k < P; ++k) w[k] = f2_both(1.f);
  auto weights = [&](int c) {
    if (a.w && c < a.cols) load_weights<W>(a.w, a.w_f32, c, w);
  };
  if (KEEP) weights(lane * W);
  // a block's rows: R times `groups` of them, one of each R for every group
  for (long long r0 = static_cast<long long>(blockIdx.x) * groups * R; r0 < a.rows; r0 += static_cast<long long>(gridDim.x) * groups * R) {
    RowVec<T> x[R][NV], g[R][NV];
    float2 st[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long row = r0 + r * groups + group;
      const bool live = row < a.rows;
      st[r] = live ? *reinterpret_cast<const float2*>(a.stats + 2 * row) : make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * lanes + lane) * W;
        if (live && c < a.cols) {
          x[r][i].load(static_cast<const T*>(a.x) + row * a.ld_x + c);
          g[r][i].load(static_cast<const T*>(a.dy) + row * a.ld_dy + c);
        }
      }
    }
    float s[2 * R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const bool live = r0 + r * groups + group < a.rows;
      const uint64_t m = f2_both(st[r].x), rs = f2_both(st[r].y);
      uint64_t s1 = 0ull, s2 = 0ull;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * lanes + lane) * W;
        if (live && c < a.cols) {
          uint64_t fx[P], fg[P];
          if (!KEEP) weights(c);
          x[r][i].get(fx);
          g[r][i].get(fg);
#pragma unroll
          for (int k = 0; k < P; ++k) {
            const uint64_t xhat = f2_mul(f2_sub(fx[k], m), rs), gw = f2_mul(fg[k], w[k]);
            dw[i][k] = f2_fma(fg[k], xhat, dw[i][k]);
            db[i][k] = f2_add(db[i][k], fg[k]);
            s1 = f2_add(s1, gw);
            s2 = f2_fma(gw, xhat, s2);
          }
        }
      }
      s[2 * r] = f2_sum(s1);
      s[2 * r + 1] = f2_sum(s2);
    }
    row_sums<BLOCK, 2 * R>(s, cut.group, part);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long row = r0 + r * groups + group;
      if (row < a.rows) {
        const uint64_t m = f2_both(st[r].x), rs = f2_both(st[r].y), m1 = f2_both(s[2 * r] * inv), m2 = f2_both(-s[2 * r + 1] * inv);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int c = (i * lanes + lane) * W;
          if (c < a.cols) {
            uint64_t fx[P], fg[P];
            if (!KEEP) weights(c);
            x[r][i].get(fx);
            g[r][i].get(fg);
#pragma unroll
            for (int k = 0; k < P; ++k) {
              const uint64_t xhat = f2_mul(f2_sub(fx[k], m), rs), gw = f2_mul(fg[k], w[k]);
              fg[k] = f2_mul(rs, f2_fma(xhat, m2, f2_sub(gw, m1)));
            }
            RowVec<T>::store(static_cast<T*>(a.y) + row * a.ld_y + c, fg);
          }
        }
      }
    }
  }
  if (!a.dw && !a.db) return;
  auto each = [&](auto&& put) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < P; ++k) {
        const int c = (i * lanes + lane) * W + 2 * k;
        float w0, w1, b0, b1;
        f2_unpack(dw[i][k], w0, w1);
        f2_unpack(db[i][k], b0, b1);
        if (c < a.cols) put(c, w0, b0);
        if (c + 1 < a.cols) put(c + 1, w1, b1);
      }
  };
  if constexpr (BLOCK) {
    float* out = FEW ? joined : a.work + static_cast<long long>(blockIdx.x) * 2 * a.cols;
    each([&](int c, float dw_, float db_) {
      out[c] = dw_;
      out[a.cols + c] = db_;
    });
    if constexpr (FEW) cluster_sums(a, joined);
  } else {
    for (int o = lanes; o < 32; o <<= 1)
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < P; ++k) {
          dw[i][k] = f2_add(dw[i][k], __shfl_xor_sync(0xffffffffu, dw[i][k], o));
          db[i][k] = f2_add(db[i][k], __shfl_xor_sync(0xffffffffu, db[i][k], o));
        }
    join_warps<FEW>(a, joined, lanes, each);
  }
}

// The same element by element, for rows that start anywhere.
template <typename T, int NV, int R, bool BLOCK, int THREADS, int MIN, bool FEW>
__global__ void __launch_bounds__(THREADS, MIN) ln_bwd_one_kernel(const AerisLayerNorm a, const LnCut cut) {
  __shared__ float part[BLOCK ? 64 * R : 1];
  extern __shared__ float joined[];
  chain_point();
  const int lanes = BLOCK ? blockDim.x : cut.group, lane = BLOCK ? threadIdx.x : threadIdx.x & (cut.group - 1);
  const int group = BLOCK ? 0 : threadIdx.x / cut.group, groups = BLOCK ? 1 : cut.rows;
  const float inv = 1.f / static_cast<float>(a.cols);
  float dw[NV], db[NV], w[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = i * lanes + lane;
    dw[i] = db[i] = 0.f;
    w[i] = c >= a.cols ? 0.f : a.w ? weight_at(a.w, a.w_f32, c) : 1.f;
  }
  for (long long r0 = static_cast<long long>(blockIdx.x) * groups * R; r0 < a.rows; r0 += static_cast<long long>(gridDim.x) * groups * R) {
    T x[R][NV], g[R][NV];
    float2 st[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long row = r0 + r * groups + group;
      const bool live = row < a.rows;
      st[r] = live ? *reinterpret_cast<const float2*>(a.stats + 2 * row) : make_float2(0.f, 0.f);
      const T *px = static_cast<const T*>(a.x) + row * a.ld_x + lane, *pg = static_cast<const T*>(a.dy) + row * a.ld_dy + lane;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const bool in = live && i * lanes + lane < a.cols;
        x[r][i] = in ? px[i * lanes] : T(0.f);
        g[r][i] = in ? pg[i * lanes] : T(0.f);
      }
    }
    float s[2 * R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      s[2 * r] = s[2 * r + 1] = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        // zeros of dy behind the row's end add nothing; the statistics there are finite
        const float xhat = (ld_f(&x[r][i]) - st[r].x) * st[r].y, fg = ld_f(&g[r][i]), gw = fg * w[i];
        dw[i] = fmaf(fg, xhat, dw[i]);
        db[i] += fg;
        s[2 * r] += gw;
        s[2 * r + 1] = fmaf(gw, xhat, s[2 * r + 1]);
      }
    }
    row_sums<BLOCK, 2 * R>(s, cut.group, part);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long row = r0 + r * groups + group;
      if (row < a.rows) {
        const float m1 = s[2 * r] * inv, m2 = s[2 * r + 1] * inv;
        T* dx = static_cast<T*>(a.y) + row * a.ld_y + lane;
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if (i * lanes + lane < a.cols) {
            const float xhat = (ld_f(&x[r][i]) - st[r].x) * st[r].y;
            st_f(dx + i * lanes, st[r].y * (fmaf(ld_f(&g[r][i]), w[i], -m1) - xhat * m2));
          }
      }
    }
  }
  if (!a.dw && !a.db) return;
  auto each = [&](auto&& put) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = i * lanes + lane;
      if (c < a.cols) put(c, dw[i], db[i]);
    }
  };
  if constexpr (BLOCK) {
    float* out = FEW ? joined : a.work + static_cast<long long>(blockIdx.x) * 2 * a.cols;
    each([&](int c, float dw_, float db_) {
      out[c] = dw_;
      out[a.cols + c] = db_;
    });
    if constexpr (FEW) cluster_sums(a, joined);
  } else {
    for (int o = lanes; o < 32; o <<= 1)
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        dw[i] += __shfl_xor_sync(0xffffffffu, dw[i], o);
        db[i] += __shfl_xor_sync(0xffffffffu, db[i], o);
      }
    join_warps<FEW>(a, joined, lanes, each);
  }
}

// Rows of up to 16 K elements for a block of 1,024 threads: they are read twice, the second time from L1, for what stays in registers are
// the column sums. 201 x 12,540 bf16, which starts anywhere: 17 us and the slices' join; sums and rows in passes of their own 32.
template <typename T>
__global__ void __launch_bounds__(1024, 1) ln_bwd_long_kernel(const AerisLayerNorm a) {
  constexpr int NV = 16;
  __shared__ float part[64];
  chain_point();
  const float inv = 1.f / static_cast<float>(a.cols);
  float dw[NV], db[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) dw[i] = db[i] = 0.f;
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *x = static_cast<const T*>(a.x) + row * a.ld_x, *dy = static_cast<const T*>(a.dy) + row * a.ld_dy;
    const float2 t = *reinterpret_cast<const float2*>(a.stats + 2 * row);
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = i * 1024 + threadIdx.x;
      if (c < a.cols) {
        const float g = ld_f(dy + c), xhat = (ld_f(x + c) - t.x) * t.y, gw = a.w ? g * weight_at(a.w, a.w_f32, c) : g;
        dw[i] = fmaf(g, xhat, dw[i]);
        db[i] += g;
        s[0] += gw;
        s[1] = fmaf(gw, xhat, s[1]);
      }
    }
    row_sums<true, 2>(s, 0, part);
    const float m1 = s[0] * inv, m2 = s[1] * inv;
    T* dx = static_cast<T*>(a.y) + row * a.ld_y;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = i * 1024 + threadIdx.x;
      if (c < a.cols) {
        const float g = ld_f(dy + c), xhat = (ld_f(x + c) - t.x) * t.y, gw = a.w ? g * weight_at(a.w, a.w_f32, c) : g;
        st_f(dx + c, t.y * (gw - m1 - xhat * m2));
      }
    }
  }
  if (!a.work) return;
  float* out = a.work + static_cast<long long>(blockIdx.x) * 2 * a.cols;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = i * 1024 + threadIdx.x;
    if (c < a.cols) {
      out[c] = dw[i];
      out[a.cols + c] = db[i];
    }
  }
}

// Many rows that start anywhere: a block per R rows, which come through a ring of bulk copies some rounds ahead, in the granules of 16
// bytes that hold them (a granule with one byte of an allocation lies in it as a whole). A thread has columns threadIdx,
// threadIdx + TH, .. of all rows; weights and column sums stay in registers. More rows a round hide the
// block's sums, fewer leave registers (gradients of rows of 3,411 bf16: two rows a round 158 us, with spills, one 123). What bounds it
// is issue slots: an element at a time, of two bytes. Forward and gradients, in us, against lanes that read memory themselves:
// 19,366 x 3,411 bf16 88 and 123 (222 and 224), 50,000 x 1,001 bf16 78 and 99 (128 and 157), 20,000 x 333 fp32 17 and 23 (26 and 26),
// 1,200 x 1,001 bf16 5.3 and 6.2 (6.2 and 7.7).
struct OddRing {
  static __device__ __forceinline__ uint32_t granules(const void* row, int size) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(row);
    return static_cast<uint32_t>(((at + size + 15) & ~uintptr_t(15)) - (at & ~uintptr_t(15)));
  }
  static __device__ __forceinline__ void request(uint8_t* dst, const void* row, int size, uint64_t* bar) {
    bulk_load(dst, reinterpret_cast<const void*>(reinterpret_cast<uintptr_t>(row) & ~uintptr_t(15)), granules(row, size), bar);
  }
};
// A wait gave up: the rounds that were asked for from (st, ph) on are let in (bounded) before the block's memory is another's.
__device__ __forceinline__ void odd_drain(uint64_t* bars, int stages, int st, uint32_t ph, long long r0, long long step,
                                          const AerisLayerNorm& a) {
  for (int i = 0; i < stages && r0 < a.rows; ++i, r0 += step) {
    if (threadIdx.x < 32) mbar_wait_warp(bars + st, ph, a.status, ERR_TIMEOUT_FULL);
    if (++st == stages) { st = 0; ph ^= 1; }
  }
}
// Sums over the block in every thread; false where a thread of it says so.
template <int K>
__device__ __forceinline__ bool odd_sums(float (&v)[K], bool ok, float* part) {
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = warp_sum(v[k]);
  // everyone has taken the words of the sums before, and its elements of these rows
  if (!__syncthreads_and(ok)) return false;
  if ((threadIdx.x & 31) == 0)
#pragma unroll
    for (int k = 0; k < K; ++k) part[k * 32 + (threadIdx.x >> 5)] = v[k];
  __syncthreads();
  const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = warp_sum(lane < warps ? part[k * 32 + lane] : 0.f);
  return true;
}

template <typename T, int NV, int R, int TH>
__global__ void __launch_bounds__(TH, 1024 / TH) ln_fwd_odd_kernel(const AerisLayerNorm a, const int stages, const int bytes) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float part[32 * R];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem);
  uint8_t* mem = smem + 64;
  if (threadIdx.x == 0) {
    for (int i = 0; i < stages; ++i) mbar_init(bars + i, 1);
    fence_barrier_init();
  }
  __syncthreads();
  chain_point();
  const int size = a.cols * static_cast<int>(sizeof(T));
  const T* x0 = static_cast<const T*>(a.x);
  const long long step = static_cast<long long>(gridDim.x) * R;
  auto request = [&](long long r0, int st) {
    if (threadIdx.x != 0 || r0 >= a.rows) return;
    uint32_t all = 0;
    for (int r = 0; r < R && r0 + r < a.rows; ++r) all += OddRing::granules(x0 + (r0 + r) * a.ld_x, size);
    mbar_expect_tx(bars + st, all);
    for (int r = 0; r < R && r0 + r < a.rows; ++r)
      OddRing::request(mem + (st * R + r) * bytes, x0 + (r0 + r) * a.ld_x, size, bars + st);
  };
  long long r0 = static_cast<long long>(blockIdx.x) * R;
  for (int i = 0; i < stages; ++i) request(r0 + i * step, i);
  float w[NV], b[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = i * TH + threadIdx.x;
    w[i] = c < a.cols && a.w ? weight_at(a.w, a.w_f32, c) : 1.f;
    b[i] = c < a.cols && a.b ? weight_at(a.b, a.w_f32, c) : 0.f;
  }
  const float inv = 1.f / static_cast<float>(a.cols);
  uint32_t ph = 0;
  for (int st = 0; r0 < a.rows; r0 += step) {
    const bool ok = mbar_wait_warp(bars + st, ph, a.status, ERR_TIMEOUT_FULL);
    float v[R][NV], s[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const T* x = reinterpret_cast<const T*>(mem + (st * R + r) * bytes + (reinterpret_cast<uintptr_t>(x0 + (r0 + r) * a.ld_x) & 15));
      s[r] = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = i * TH + threadIdx.x;
        v[r][i] = c < a.cols && r0 + r < a.rows ? ld_f(x + c) : 0.f;
        s[r] += v[r][i];
      }
    }
    if (!odd_sums(s, ok, part)) {
      odd_drain(bars, stages, st, ph, r0, step, a);
      return;
    }
    request(r0 + stages * step, st);
    if (++st == stages) { st = 0; ph ^= 1; }
    float mean[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      mean[r] = s[r] * inv;
      s[r] = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        v[r][i] -= mean[r];
        if (i * TH + static_cast<int>(threadIdx.x) < a.cols) s[r] = fmaf(v[r][i], v[r][i], s[r]);
      }
    }
    odd_sums(s, true, part);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (r0 + r >= a.rows) continue;
      const float rstd = 1.f / sqrtf(s[r] * inv + a.eps);
      T* y = static_cast<T*>(a.y) + (r0 + r) * a.ld_y;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = i * TH + threadIdx.x;
        if (c < a.cols) st_f(y + c, fmaf(v[r][i] * rstd, w[i], b[i]));
      }
      if (threadIdx.x == 0) *reinterpret_cast<float2*>(a.stats + 2 * (r0 + r)) = make_float2(mean[r], rstd);
    }
  }
}

template <typename T, int NV, int R, int TH>
__global__ void __launch_bounds__(TH, 1024 / TH) ln_bwd_odd_kernel(const AerisLayerNorm a, const int stages, const int bytes) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float part[64 * R];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem);
  uint8_t* mem = smem + 64;
  if (threadIdx.x == 0) {
    for (int i = 0; i < stages; ++i) mbar_init(bars + i, 1);
    fence_barrier_init();
  }
  __syncthreads();
  chain_point();
  const int size = a.cols * static_cast<int>(sizeof(T));
  const T *x0 = static_cast<const T*>(a.x), *g0 = static_cast<const T*>(a.dy);
  const long long step = static_cast<long long>(gridDim.x) * R;
  auto request = [&](long long r0, int st) {
    if (threadIdx.x != 0 || r0 >= a.rows) return;
    uint32_t all = 0;
    for (int r = 0; r < R && r0 + r < a.rows; ++r)
      all += OddRing::granules(x0 + (r0 + r) * a.ld_x, size) + OddRing::granules(g0 + (r0 + r) * a.ld_dy, size);
    mbar_expect_tx(bars + st, all);
    for (int r = 0; r < R && r0 + r < a.rows; ++r) {
      uint8_t* dst = mem + (st * R + r) * 2 * bytes;
      OddRing::request(dst, x0 + (r0 + r) * a.ld_x, size, bars + st);
      OddRing::request(dst + bytes, g0 + (r0 + r) * a.ld_dy, size, bars + st);
    }
  };
  long long r0 = static_cast<long long>(blockIdx.x) * R;
  for (int i = 0; i < stages; ++i) request(r0 + i * step, i);
  float w[NV], dw[NV], db[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = i * TH + threadIdx.x;
    w[i] = c < a.cols && a.w ? weight_at(a.w, a.w_f32, c) : 1.f;
    dw[i] = db[i] = 0.f;
  }
  const float inv = 1.f / static_cast<float>(a.cols);
  uint32_t ph = 0;
  for (int st = 0; r0 < a.rows; r0 += step) {
    const bool ok = mbar_wait_warp(bars + st, ph, a.status, ERR_TIMEOUT_FULL);
    float v[R][NV], g[R][NV], s[2 * R];       // v: xhat
    float rstd[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const bool live = r0 + r < a.rows;
      const float2 t = live ? *reinterpret_cast<const float2*>(a.stats + 2 * (r0 + r)) : make_float2(0.f, 0.f);
      const uint8_t* at = mem + (st * R + r) * 2 * bytes;
      const T* x = reinterpret_cast<const T*>(at + (reinterpret_cast<uintptr_t>(x0 + (r0 + r) * a.ld_x) & 15));
      const T* dy = reinterpret_cast<const T*>(at + bytes + (reinterpret_cast<uintptr_t>(g0 + (r0 + r) * a.ld_dy) & 15));
      rstd[r] = t.y;
      s[2 * r] = s[2 * r + 1] = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = i * TH + threadIdx.x;
        const bool in = c < a.cols && live;
        v[r][i] = in ? (ld_f(x + c) - t.x) * t.y : 0.f;
        const float d = in ? ld_f(dy + c) : 0.f;
        dw[i] = fmaf(d, v[r][i], dw[i]);
        db[i] += d;
        g[r][i] = d * w[i];
        s[2 * r] += g[r][i];
        s[2 * r + 1] = fmaf(g[r][i], v[r][i], s[2 * r + 1]);
      }
    }
    if (!odd_sums(s, ok, part)) {
      odd_drain(bars, stages, st, ph, r0, step, a);
      return;
    }
    request(r0 + stages * step, st);
    if (++st == stages) { st = 0; ph ^= 1; }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (r0 + r >= a.rows) continue;
      const float m1 = s[2 * r] * inv, m2 = s[2 * r + 1] * inv;
      T* dx = static_cast<T*>(a.y) + (r0 + r) * a.ld_y;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = i * TH + threadIdx.x;
        if (c < a.cols) st_f(dx + c, rstd[r] * (g[r][i] - m1 - v[r][i] * m2));
      }
    }
  }
  if (!a.work) return;
  float* out = a.work + static_cast<long long>(blockIdx.x) * 2 * a.cols;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = i * TH + threadIdx.x;
    if (c < a.cols) {
      out[c] = dw[i];
      out[a.cols + c] = db[i];
    }
  }
}

// `slices`: null forward; backward it receives how many slices of column sums were written.
template <typename T, int NV, int RF, int RB, int TH>
int launch_ln_odd(const AerisLayerNorm& a, cudaStream_t stream, int* slices) {
  constexpr int PER_SM = 1024 / TH;
  const int R = slices ? RB : RF;
  const int bytes = (a.cols * static_cast<int>(sizeof(T)) + 30) / 16 * 16, row = slices ? 2 * bytes : bytes;
  // three at least, but for the widest fp32 rows of 64 and of 128 threads (241 to 256, 509 to 512 columns): two
  int stages = (200 * 1024 / PER_SM - 1024) / (R * row);
  if (stages > 6) stages = 6;
  const long long need = (a.rows + R - 1) / R;
  long long blocks = static_cast<long long>(num_sms()) * PER_SM;
  if (blocks > need) blocks = need;
  if (slices && a.work && blocks > a.slices) blocks = a.slices;
  const int smem = 64 + stages * R * row;
  if (slices) {
    static std::atomic<uint64_t> done{0};
    if (!allow_smem_once(ln_bwd_odd_kernel<T, NV, RB, TH>, 200 * 1024, done)) return -20;
    *slices = static_cast<int>(blocks);
    return launch_chained(ln_bwd_odd_kernel<T, NV, RB, TH>, static_cast<unsigned>(blocks), TH, smem, stream, a, stages, bytes);
  }
  static std::atomic<uint64_t> done{0};
  if (!allow_smem_once(ln_fwd_odd_kernel<T, NV, RF, TH>, 200 * 1024, done)) return -20;
  return launch_chained(ln_fwd_odd_kernel<T, NV, RF, TH>, static_cast<unsigned>(blocks), TH, smem, stream, a, stages, bytes);
}
// Where rows are many enough for rounds that follow one another; others, and the widest, go straight from memory (returns 1).
template <typename T>
int ln_odd(const AerisLayerNorm& a, cudaStream_t stream, int* slices) {
  if (a.rows < 8 * num_sms() || a.cols <= 96 || a.cols > 8192) return 1;
  if (a.cols <= 256) return launch_ln_odd<T, 4, 4, 2, 64>(a, stream, slices);
  if (a.cols <= 512) return launch_ln_odd<T, 4, 4, 2, 128>(a, stream, slices);
  if (a.cols <= 1024) return launch_ln_odd<T, 4, 4, 2, 256>(a, stream, slices);
  if (a.cols <= 2048) return launch_ln_odd<T, 4, 4, 2, 512>(a, stream, slices);
  if (a.cols <= 4096) return launch_ln_odd<T, 8, 2, 1, 512>(a, stream, slices);
  return launch_ln_odd<T, 8, 1, 1, 1024>(a, stream, slices);
}

bool ln_aligned(const void* p, long long ld, int size) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (ld * size) % 16 == 0;
}

template <typename T, int W, int NV, bool BLOCK>
int launch_ln_fwd(const AerisLayerNorm& a, LnCut cut, int threads, cudaStream_t stream) {
  const long long blocks = BLOCK ? a.rows : (a.rows + cut.rows - 1) / cut.rows;
  if constexpr (W > 1)
    return launch_chained(ln_fwd_kernel<T, W, NV, BLOCK>, static_cast<unsigned>(blocks), threads, 0, stream, a, cut);
  else
    return launch_chained(ln_fwd_one_kernel<T, NV, BLOCK>, static_cast<unsigned>(blocks), threads, 0, stream, a, cut);
}

// The cut of rows of `vecs` vectors into lanes: groups of a warp, as many lanes as there are vectors, up to all of them.
LnCut ln_cut(int vecs) {
  LnCut c;
  c.group = 1;
  while (c.group < vecs && c.group < 32) c.group *= 2;
  c.rows = 256 / c.group;
  return c;
}
int ln_threads(int vecs, int nv) { return ((vecs + nv - 1) / nv + 31) / 32 * 32; }

// Forward. Returns 1 where no kernel takes the width.
template <typename T>
int ln_fwd_fast(const AerisLayerNorm& a, cudaStream_t stream) {
  constexpr int S = sizeof(T), W = 16 / S;
  if (a.cols % W == 0 && ln_aligned(a.x, a.ld_x, S) && ln_aligned(a.y, a.ld_y, S) && ln_aligned(a.w, 0, S) && ln_aligned(a.b, 0, S)) {
    const int vecs = a.cols / W, nv = (vecs + 31) / 32;
    const LnCut cut = ln_cut(vecs);
    // few rows: a block each, as long as that makes the chain of a row's steps shorter
    if (nv > 2 && a.rows <= 2 * num_sms() && vecs <= 1024) return launch_ln_fwd<T, W, 1, true>(a, cut, ln_threads(vecs, 1), stream);
    if (nv <= 1) return launch_ln_fwd<T, W, 1, false>(a, cut, 256, stream);
    if (nv <= 2) return launch_ln_fwd<T, W, 2, false>(a, cut, 256, stream);
    if (nv <= 4) return launch_ln_fwd<T, W, 4, false>(a, cut, 256, stream);
    if (nv <= 6) return launch_ln_fwd<T, W, 6, false>(a, cut, 256, stream);
    if (nv <= 8) return launch_ln_fwd<T, W, 8, false>(a, cut, 256, stream);
    if (vecs <= 2048) return launch_ln_fwd<T, W, 2, true>(a, cut, ln_threads(vecs, 2), stream);
    if (vecs <= 4096) return launch_ln_fwd<T, W, 4, true>(a, cut, ln_threads(vecs, 4), stream);
    return 1;
  }
  const int odd = ln_odd<T>(a, stream, nullptr);
  if (odd <= 0) return odd;
  const int nv = (a.cols + 31) / 32;
  const LnCut cut = ln_cut(a.cols);
  if (nv <= 1) return launch_ln_fwd<T, 1, 1, false>(a, cut, 256, stream);
  if (nv <= 2) return launch_ln_fwd<T, 1, 2, false>(a, cut, 256, stream);
  if (nv <= 4) return launch_ln_fwd<T, 1, 4, false>(a, cut, 256, stream);
  if (nv <= 8) return launch_ln_fwd<T, 1, 8, false>(a, cut, 256, stream);
  if (nv <= 16) return launch_ln_fwd<T, 1, 16, false>(a, cut, 256, stream);
  if (a.cols <= 8192) return launch_ln_fwd<T, 1, 8, true>(a, cut, ln_threads(a.cols, 8), stream);
  if (a.cols <= 16384) return launch_ln_fwd<T, 1, 16, true>(a, cut, ln_threads(a.cols, 16), stream);
  return 1;
}

// `slices`: receives how many slices of column sums were written.
template <typename T, int W, int NV, int R, bool BLOCK, int THREADS, int MIN>
int launch_ln_bwd(const AerisLayerNorm& a, LnCut cut, int threads, cudaStream_t stream, int& slices) {
  const int at_once = (BLOCK ? 1 : cut.rows) * R;       // rows of a block
  const long long need = (a.rows + at_once - 1) / at_once;
  // as many blocks as the SMs hold (MIN, more of narrower ones)
  long long blocks = static_cast<long long>(num_sms()) * (MIN * THREADS / threads);
  if (blocks > need) blocks = need;
  const bool sums = a.dw || a.db;
  const bool cluster = sums && !a.work;
  if (cluster) {
    blocks = 1;
    while (2 * blocks <= need && blocks < 8) blocks *= 2;
  } else if (sums && blocks > a.slices) {
    blocks = a.slices;
  }
  slices = static_cast<int>(blocks);
  const int smem = sums && (!BLOCK || cluster) ? 2 * a.cols * 4 : 0;
  const auto kernel = [](auto few) {
    if constexpr (W > 1) return ln_bwd_kernel<T, W, NV, R, BLOCK, THREADS, MIN, few.value>;
    else return ln_bwd_one_kernel<T, NV, R, BLOCK, THREADS, MIN, few.value>;
  };
  return cluster ? launch_chained_cluster(kernel(std::true_type{}), slices, threads, smem, stream, a, cut)
                 : launch_chained(kernel(std::false_type{}), slices, threads, smem, stream, a, cut);
}
template <typename T>
int ln_bwd_fast(const AerisLayerNorm& a, cudaStream_t stream, int& slices) {
  constexpr int S = sizeof(T), W = 16 / S;
  if (a.cols % W == 0 && ln_aligned(a.x, a.ld_x, S) && ln_aligned(a.y, a.ld_y, S) && ln_aligned(a.dy, a.ld_dy, S) && ln_aligned(a.w, 0, S)) {
    const int vecs = a.cols / W;
    const LnCut cut = ln_cut(vecs);
    if (vecs <= 32) return launch_ln_bwd<T, W, 1, 4, false, 256, 2>(a, cut, 256, stream, slices);
    if (vecs <= 64) return launch_ln_bwd<T, W, 2, 2, false, 256, 2>(a, cut, 256, stream, slices);
    if (vecs <= 192) return launch_ln_bwd<T, W, 1, 4, true, 192, 3>(a, cut, ln_threads(vecs, 1), stream, slices);
    if (vecs <= 256) return launch_ln_bwd<T, W, 1, 4, true, 256, 2>(a, cut, ln_threads(vecs, 1), stream, slices);
    // Two blocks an SM, or one of 1,024 threads: 14,400 x 2560 bf16 78 -> 61 us, x 4096 96 -> 90, 7,200 x 12288 192 -> 166, against one of 512
    // with more rows at a time. Two vectors a thread suit fp32, whose vectors are half as many elements: 14,400 x 2048 70 us, with
    // one 85; bf16 14,400 x 4096 97 and 90.
    if (vecs <= 512) {
      if constexpr (W == 4) return launch_ln_bwd<T, W, 2, 2, true, 256, 2>(a, cut, ln_threads(vecs, 2), stream, slices);
      else return launch_ln_bwd<T, W, 1, 2, true, 512, 2>(a, cut, ln_threads(vecs, 1), stream, slices);
    }
    if (vecs <= 1024) return launch_ln_bwd<T, W, 1, 2, true, 1024, 1>(a, cut, ln_threads(vecs, 1), stream, slices);
    if (vecs <= 2048) return launch_ln_bwd<T, W, 2, 1, true, 1024, 1>(a, cut, ln_threads(vecs, 2), stream, slices);
    return 1;
  }
  if ((!a.dw && !a.db) || a.work) {
    const int odd = ln_odd<T>(a, stream, &slices);
    if (odd <= 0) return odd;
  }
  const LnCut cut = ln_cut(a.cols);
  if (a.cols <= 32) return launch_ln_bwd<T, 1, 1, 4, false, 256, 3>(a, cut, 256, stream, slices);
  if (a.cols <= 128) return launch_ln_bwd<T, 1, 4, 4, false, 256, 2>(a, cut, 256, stream, slices);
  if (a.cols <= 512) return launch_ln_bwd<T, 1, 4, 4, true, 128, 5>(a, cut, ln_threads(a.cols, 4), stream, slices);
  if (a.cols <= 1024) return launch_ln_bwd<T, 1, 4, 4, true, 256, 2>(a, cut, ln_threads(a.cols, 4), stream, slices);
  if (a.cols <= 4096) return launch_ln_bwd<T, 1, 8, 2, true, 512, 1>(a, cut, ln_threads(a.cols, 8), stream, slices);
  if (a.cols <= 8192) return launch_ln_bwd<T, 1, 16, 1, true, 512, 1>(a, cut, ln_threads(a.cols, 16), stream, slices);
  if (a.cols <= 16384) {
    long long blocks = num_sms();
    if (blocks > a.rows) blocks = a.rows;
    if (a.work && blocks > a.slices) blocks = a.slices;
    slices = static_cast<int>(blocks);
    return launch_chained(ln_bwd_long_kernel<T>, slices, 1024, 0, stream, a);
  }
  return 1;
}

}  // namespace

}  // namespace aeris
