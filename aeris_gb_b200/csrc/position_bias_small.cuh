// Attention with a position bias in windows of at most 96 tokens, forward and backward. Included by position_bias.cu.
//
// A tile of the fifth-generation tensor core has 128 rows, of which such a window fills an eighth to three quarters, and a tile's way
// through its pipeline takes 2 us whatever is in it. Here a warp has 16 queries, a group of warps a window and head; products are
// warp-level ones (m16n8k16), scores never leave registers, and rows of all keys are at hand, so that the softmax takes no running
// statistics. A CTA takes windows of one head, one after the other, whose bias by relative position (at most 345 entries) lies in
// shared memory. Backward everything comes from one pass: delta is the row sum of p dp (o is not read), dS is added up over the
// CTA's windows in registers, and only its sums by relative position leave the CTA.
//
// What bounds it is latency: a CTA waits for a window, works on it and waits for the next, with others of the SM in between. us in a
// graph against the kernels of large windows, forward / backward with the table's gradient: 2,000 windows of 4 x 4, 16 heads of 64,
// 56 / 98 (256 / 1,393; their bytes take 40 / 80); 500 of 6 x 5, 8 heads of 64, 19 / 40 (35 / 214); 1,000 of 8 x 8, 4 heads of 32,
// 30 / 58 (39 / 205); 1,440 of 17 x 4, one head of 72, 24 / 67 (31 / 176); 500 of 9 x 10, 4 heads of 64, 38 / 130 (34 / 148); 500 of
// 9 x 8, 4 heads of 128, 56 / 190 (50 / 241). Backward, eight sixteens of queries would not have scores, dP and sums in registers.
#pragma once

namespace aeris {

namespace {

constexpr int SMALL_MOST = 200 * 1024;      // dynamic shared memory
constexpr int SMALL_TOKENS = 96, SMALL_HEAD = (384 + SMALL_TOKENS) * 4;       // bytes: entries of the bias, places of the tokens

struct SmallParams {
  const __nv_bfloat16 *qkv, *d_o;
  __nv_bfloat16 *o, *dqkv;
  float *lse, *part;          // part: [runs, positions, heads]; null: not wanted
  long long ld, ldo, ldg;
  int n_win, n, d, runs, stages;
  float scale;
  BiasSource source;          // pitch: 2 wide - 1
};

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}

// NT: sixteens of tokens = warps of a window; GROUPS windows of a CTA at a time.
template <int NT> struct SmallCfg {
  static constexpr int GROUPS = NT == 1 ? 4 : NT == 2 ? 2 : 1, THREADS = GROUPS * NT * 32, ROWS = 16 * NT;
  // CTAs on an SM, as far as registers go
  static constexpr int HELD_FWD = NT == 1 ? 10 : NT == 2 ? 8 : NT == 3 ? 7 : NT == 4 ? 6 : NT == 5 ? 4 : 3;
  static constexpr int HELD_BWD = NT == 1 ? 7 : NT <= 3 ? 5 : NT == 4 ? 3 : NT == 5 ? 2 : 1;
  static constexpr int P_PITCH = ROWS * 2 + 16;      // odd in 16-byte units, as the operands' pitch: eight rows are in different banks
  static __host__ __device__ __forceinline__ int pitch(int d) { return (d + 15) / 16 * 32 + 16; }
  // a group's: operands of one or two windows, and backward P and dS
  static __host__ __device__ __forceinline__ int stage_bytes(int d, bool backward) { return (backward ? 4 : 3) * ROWS * pitch(d); }
  static __host__ __device__ __forceinline__ int group_bytes(int d, bool backward, int stages) {
    return stages * stage_bytes(d, backward) + (backward ? 2 * ROWS * P_PITCH : 0);
  }
  static __host__ __device__ __forceinline__ int bytes(int d, bool backward, int stages) {
    return SMALL_HEAD + GROUPS * group_bytes(d, backward, stages);
  }
  static int held(int d, bool backward, int stages) {
    const int by_memory = 228 * 1024 / (bytes(d, backward, stages) + 1024), most = backward ? HELD_BWD : HELD_FWD;
    return by_memory < most ? by_memory : most;
  }
  // Two where three CTAs still fit on an SM: 2,000 windows of 4 x 4, 16 heads of 64, 68 -> 56 us forward (four CTAs for eight), but
  // backward with two CTAs for five 1.9 times as long; 1,000 of 8 x 8, 4 heads: of 64 47 -> 36 forward (three for six), of 128 67 -> 72 (two for four).
  static int stages(int d, bool backward) { return held(d, backward, 2) >= 3 ? 2 : 1; }
};

// What a warp knows of its CTA, group and lanes.
template <int NT> struct SmallWarp {
  using C = SmallCfg<NT>;
  const SmallParams& p;
  uint8_t *mem, *next;      // the group's operands: of the window at hand and, where there is room, of the next one
  float* bias;
  int* at;                  // places, of the last token from the window's end on
  uint8_t* scores_mem;      // backward: P, behind it dS
  int head, group, wq, lane, t, pitch;      // wq: which sixteen of the queries; t: thread of the group
  int r0, c0, dr, dc;       // this thread's first 16 bytes of a window's rows, and from one to the next

  __device__ __forceinline__ void barrier() const {
    if constexpr (NT == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(NT * 32) : "memory");
  }
  __device__ __forceinline__ uint32_t tile(int which) const { return smem_u32(mem) + which * C::ROWS * pitch; }
  // rows [n, d] of a window to operand tile `which` of those at `to`
  __device__ __forceinline__ void load(const uint8_t* to, int which, const __nv_bfloat16* src, long long ld) const {
    const int per = p.d / 8;
    const uint32_t dst = smem_u32(to) + which * C::ROWS * pitch;
    for (int r = r0, c = c0; r < p.n; r += dr, c += dc) {
      if (c >= per) {
        c -= per;
        if (++r >= p.n) break;
      }
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + r * pitch + c * 16), "l"(src + r * ld + c * 8) : "memory");
    }
  }
  __device__ __forceinline__ void loaded() const {
    asm volatile("cp.async.wait_all;" ::: "memory");
    barrier();
  }
  __device__ __forceinline__ void turn() {
    uint8_t* m = mem;
    mem = next;
    next = m;
  }
  // this warp's sixteen rows of tile `which` to memory
  __device__ __forceinline__ void store(int which, __nv_bfloat16* dst, long long ld) const {
    __syncwarp();
    const int per = p.d / 8, rows = min(16, p.n - 16 * wq);
    const uint8_t* src = mem + which * C::ROWS * pitch + 16 * wq * pitch;
    for (int i = lane; i < rows * per; i += 32) {
      const int r = i / per, c = i - r * per;
      *reinterpret_cast<uint4*>(dst + (16 * wq + r) * ld + c * 8) = *reinterpret_cast<const uint4*>(src + r * pitch + c * 16);
    }
    __syncwarp();
  }
  // s[16 queries x all keys] = rows of tile `a` x (rows of tile `b`)^T
  __device__ __forceinline__ void scores(float (&s)[2 * NT][4], int a, int b) const {
#pragma unroll
    for (int i = 0; i < 2 * NT; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) s[i][k] = 0.f;
    const uint32_t pa = tile(a) + (16 * wq + (lane & 15)) * pitch + (lane >> 4) * 16;
    const uint32_t pb = tile(b) + ((lane & 7) + ((lane >> 4) << 3)) * pitch + ((lane >> 3) & 1) * 16;
    for (int c = 0; c < (p.d + 15) / 16; ++c) {
      uint32_t fa[4];
      ldsm4(fa, pa + c * 32);
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        uint32_t fb[4];
        ldsm4(fb, pb + 16 * j * pitch + c * 32);
        mma16(s[2 * j], fa, fb[0], fb[1]);
        mma16(s[2 * j + 1], fa, fb[2], fb[3]);
      }
    }
  }
  // this warp's rows of tile `to` = f (16 rows x all) x tile `b`, times `f0`, `f1` (the row's and that of the row eight further).
  // Rows and columns past the window's are left: zeros, whatever products of them would be.
  __device__ __forceinline__ void product(const uint32_t (&f)[NT][4], int b, int to, float f0, float f1) const {
    const uint32_t pb = tile(b) + (lane & 15) * pitch + (lane >> 4) * 16;
    uint8_t* out = mem + to * C::ROWS * pitch + (16 * wq + (lane >> 2)) * pitch + (lane & 3) * 4;
    const int row = 16 * wq + (lane >> 2);
    for (int c = 0; c < (p.d + 15) / 16; ++c) {
      float acc[2][4] = {};
#pragma unroll
      for (int k = 0; k < NT; ++k) {
        uint32_t fb[4];
        ldsm4_t(fb, pb + 16 * k * pitch + c * 32);
        mma16(acc[0], f[k], fb[0], fb[1]);
        mma16(acc[1], f[k], fb[2], fb[3]);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (16 * c + 8 * h < p.d) {
          if (row < p.n) *reinterpret_cast<uint32_t*>(out + c * 32 + h * 16) = pack_bf16x2(acc[h][0] * f0, acc[h][1] * f0);
          if (row + 8 < p.n) *reinterpret_cast<uint32_t*>(out + 8 * pitch + c * 32 + h * 16) = pack_bf16x2(acc[h][2] * f1, acc[h][3] * f1);
        }
    }
  }
  // scores in log2 units with their biases; -infinity past the window's keys
  __device__ __forceinline__ void biased(float (&s)[2 * NT][4]) const {
    const float sl = p.scale * 1.4426950408889634f;
    const int zero = at[p.n - 1], i0 = 16 * wq + (lane >> 2);
    const float *b0 = bias + zero + at[i0], *b1 = bias + zero + at[i0 + 8];
#pragma unroll
    for (int i = 0; i < 2 * NT; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int j = 8 * i + 2 * (lane & 3) + e, a = at[j];
        s[i][e] = j < p.n ? fmaf(s[i][e], sl, b0[-a]) : -INFINITY;
        s[i][2 + e] = j < p.n ? fmaf(s[i][2 + e], sl, b1[-a]) : -INFINITY;
      }
  }
};

template <int NT>
__device__ __forceinline__ SmallWarp<NT> small_warp(const SmallParams& p, uint8_t* smem, bool backward) {
  using C = SmallCfg<NT>;
  const int group = threadIdx.x / (NT * 32), t = threadIdx.x - group * NT * 32;
  float* bias = reinterpret_cast<float*>(smem);
  int* at = reinterpret_cast<int*>(bias + 384);
  for (int i = threadIdx.x; i < SMALL_TOKENS; i += C::THREADS) at[i] = p.source.at(min(i, p.n - 1));
  // zeros where operands end: nothing else is written there
  const int bytes = C::group_bytes(p.d, backward, p.stages), stage = C::stage_bytes(p.d, backward);
  for (int i = threadIdx.x; i < C::GROUPS * bytes / 16; i += C::THREADS)
    reinterpret_cast<uint4*>(smem + SMALL_HEAD)[i] = make_uint4(0, 0, 0, 0);
  __syncthreads();
  uint8_t* mem = smem + SMALL_HEAD + group * bytes;
  const int per = p.d / 8;
  return {p, mem, mem + (p.stages - 1) * stage, bias, at, mem + p.stages * stage, static_cast<int>(blockIdx.x), group, t >> 5,
          static_cast<int>(threadIdx.x & 31), t, C::pitch(p.d), t / per, t % per, NT * 32 / per, NT * 32 % per};
}
template <int NT>
__device__ __forceinline__ void small_table(const SmallWarp<NT>& w) {
  const int size = (2 * w.p.source.high - 1) * w.p.source.pitch;
  for (int i = threadIdx.x; i < size; i += SmallCfg<NT>::THREADS) w.bias[i] = w.p.source.entry(i, w.head);
}

template <int NT>
__global__ void __launch_bounds__(SmallCfg<NT>::THREADS, SmallCfg<NT>::HELD_FWD) small_fwd_kernel(const SmallParams p) {
  using C = SmallCfg<NT>;
  extern __shared__ __align__(16) uint8_t smem[];
  SmallWarp<NT> w = small_warp<NT>(p, smem, false);
  chain_point();
  const int heads = p.source.heads, inner = heads * p.d, step = p.runs * C::GROUPS;
  auto load = [&](int win, const uint8_t* to) {
    if (win >= p.n_win) return;
    const __nv_bfloat16* rows = p.qkv + static_cast<long long>(win) * p.n * p.ld + w.head * p.d;
#pragma unroll
    for (int i = 0; i < 3; ++i) w.load(to, i, rows + i * inner, p.ld);
  };
  int win = blockIdx.y * C::GROUPS + w.group;
  load(win, w.mem);
  small_table(w);
  __syncthreads();
  for (; win < p.n_win; win += step) {
    w.loaded();
    if (p.stages == 2) load(win + step, w.next);
    float s[2 * NT][4];
    w.scores(s, 0, 1);
    w.biased(s);
    float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
    for (int i = 0; i < 2 * NT; ++i) {
      m0 = fmaxf(m0, fmaxf(s[i][0], s[i][1]));
      m1 = fmaxf(m1, fmaxf(s[i][2], s[i][3]));
    }
    m0 = quad_max(m0);
    m1 = quad_max(m1);
    if (m0 == -INFINITY) m0 = 0.f;        // sees nothing: every term is zero
    if (m1 == -INFINITY) m1 = 0.f;
    float l0 = 0.f, l1 = 0.f;
#pragma unroll
    for (int i = 0; i < 2 * NT; ++i) {
      s[i][0] = bg_exp2(s[i][0] - m0);
      s[i][1] = bg_exp2(s[i][1] - m0);
      s[i][2] = bg_exp2(s[i][2] - m1);
      s[i][3] = bg_exp2(s[i][3] - m1);
      l0 += s[i][0] + s[i][1];
      l1 += s[i][2] + s[i][3];
    }
    l0 = quad_sum(l0);
    l1 = quad_sum(l1);
    // p leaves for the product in bf16, half a step of it at most (2^-8); the row sums are those of fp32
    uint32_t f[NT][4];
#pragma unroll
    for (int k = 0; k < NT; ++k)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        f[k][2 * h] = pack_bf16x2(s[2 * k + h][0], s[2 * k + h][1]);
        f[k][2 * h + 1] = pack_bf16x2(s[2 * k + h][2], s[2 * k + h][3]);
      }
    __syncwarp();
    w.product(f, 2, 0, l0 == 0.f ? 0.f : 1.f / l0, l1 == 0.f ? 0.f : 1.f / l1);       // this warp alone has read these queries
    w.store(0, p.o + static_cast<long long>(win) * p.n * p.ldo + w.head * p.d, p.ldo);
    float* lse = p.lse + (static_cast<long long>(win) * heads + w.head) * p.n;
    const int row = 16 * w.wq + (w.lane >> 2);
    if ((w.lane & 3) == 0) {
      if (row < p.n) lse[row] = l0 == 0.f ? INFINITY : m0 + __log2f(l0);
      if (row + 8 < p.n) lse[row + 8] = l1 == 0.f ? INFINITY : m1 + __log2f(l1);
    }
    if (p.stages == 1) {
      w.barrier();
      load(win + step, w.mem);
    }
    w.turn();
  }
}

template <int NT>
__global__ void __launch_bounds__(SmallCfg<NT>::THREADS, SmallCfg<NT>::HELD_BWD) small_bwd_kernel(const SmallParams p) {
  using C = SmallCfg<NT>;
  extern __shared__ __align__(16) uint8_t smem[];
  SmallWarp<NT> w = small_warp<NT>(p, smem, true);
  chain_point();
  const int heads = p.source.heads, inner = heads * p.d, row = 16 * w.wq + (w.lane >> 2), step = p.runs * C::GROUPS;
  uint8_t* pp = w.scores_mem;        // P, behind it dS: [queries, keys] bf16
  constexpr int P_BYTES = C::ROWS * C::P_PITCH;
  float sum[2 * NT][4];
#pragma unroll
  for (int i = 0; i < 2 * NT; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) sum[i][k] = 0.f;
  float next0 = 0.f, next1 = 0.f;       // lse of the next window's rows
  auto load = [&](int win, const uint8_t* to) {
    if (win >= p.n_win) return;
    const __nv_bfloat16* rows = p.qkv + static_cast<long long>(win) * p.n * p.ld + w.head * p.d;
#pragma unroll
    for (int i = 0; i < 3; ++i) w.load(to, i, rows + i * inner, p.ld);
    w.load(to, 3, p.d_o + static_cast<long long>(win) * p.n * p.ldo + w.head * p.d, p.ldo);
    const float* lse = p.lse + (static_cast<long long>(win) * heads + w.head) * p.n;
    if (row < p.n) next0 = lse[row];
    if (row + 8 < p.n) next1 = lse[row + 8];
  };
  int win = blockIdx.y * C::GROUPS + w.group;
  load(win, w.mem);
  small_table(w);
  __syncthreads();
  for (; win < p.n_win; win += step) {
    w.loaded();
    const float lse0 = next0, lse1 = next1;
    if (p.stages == 2) load(win + step, w.next);
    uint32_t f[NT][4];
    {
      float s[2 * NT][4], dp[2 * NT][4];
      w.scores(s, 0, 1);
      w.scores(dp, 3, 2);
      w.biased(s);
      float d0 = 0.f, d1 = 0.f;
#pragma unroll
      for (int i = 0; i < 2 * NT; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          // products past the window's rows and keys may be anything
          const bool key = 8 * i + 2 * (w.lane & 3) + e < p.n;
          s[i][e] = key && row < p.n ? bg_exp2(s[i][e] - lse0) : 0.f;
          s[i][2 + e] = key && row + 8 < p.n ? bg_exp2(s[i][2 + e] - lse1) : 0.f;
          dp[i][e] = key && row < p.n ? dp[i][e] : 0.f;
          dp[i][2 + e] = key && row + 8 < p.n ? dp[i][2 + e] : 0.f;
          d0 = fmaf(s[i][e], dp[i][e], d0);
          d1 = fmaf(s[i][2 + e], dp[i][2 + e], d1);
        }
      d0 = quad_sum(d0);
      d1 = quad_sum(d1);
      uint8_t* to = pp + row * C::P_PITCH + (w.lane & 3) * 4;
#pragma unroll
      for (int i = 0; i < 2 * NT; ++i) {
        *reinterpret_cast<uint32_t*>(to + i * 16) = pack_bf16x2(s[i][0], s[i][1]);
        *reinterpret_cast<uint32_t*>(to + 8 * C::P_PITCH + i * 16) = pack_bf16x2(s[i][2], s[i][3]);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          dp[i][e] = p.n == 1 ? 0.f : s[i][e] * (dp[i][e] - d0);          // one token sees itself whatever its score
          dp[i][2 + e] = p.n == 1 ? 0.f : s[i][2 + e] * (dp[i][2 + e] - d1);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) sum[i][k] += dp[i][k];
        const uint32_t lo = pack_bf16x2(dp[i][0], dp[i][1]), hi = pack_bf16x2(dp[i][2], dp[i][3]);
        *reinterpret_cast<uint32_t*>(to + P_BYTES + i * 16) = lo;
        *reinterpret_cast<uint32_t*>(to + P_BYTES + 8 * C::P_PITCH + i * 16) = hi;
        f[i / 2][(i & 1) * 2] = lo;
        f[i / 2][(i & 1) * 2 + 1] = hi;
      }
    }
    __nv_bfloat16* grad = p.dqkv + static_cast<long long>(win) * p.n * p.ldg + w.head * p.d;
    w.barrier();                            // P and dS are there, V has been read
    w.product(f, 1, 2, p.scale, p.scale);   // dQ = scale dS K, in V's place
    w.store(2, grad, p.ldg);
    // the transposes: this warp's sixteen keys
    auto transposed = [&](const uint8_t* m) {
      const uint32_t at = smem_u32(m) + ((w.lane & 7) + ((w.lane >> 4) << 3)) * C::P_PITCH + (16 * w.wq + ((w.lane >> 3) & 1) * 8) * 2;
#pragma unroll
      for (int k = 0; k < NT; ++k) ldsm4_t(f[k], at + 16 * k * C::P_PITCH);
    };
    transposed(pp);
    w.product(f, 3, 2, 1.f, 1.f);           // dV = P^T dO
    w.store(2, grad + 2 * inner, p.ldg);
    transposed(pp + P_BYTES);
    w.barrier();                            // K has been read
    w.product(f, 0, 1, p.scale, p.scale);   // dK = scale dS^T Q, in K's place
    w.store(1, grad + inner, p.ldg);
    if (p.stages == 1) {
      w.barrier();
      load(win + step, w.mem);
    }
    w.turn();
  }
  if (!p.part) return;
  // the groups' sums one after the other, then those by relative position
  float* all = reinterpret_cast<float*>(smem + SMALL_HEAD);
  for (int g = 0; g < C::GROUPS; ++g) {
    __syncthreads();
    if (w.group == g)
#pragma unroll
      for (int i = 0; i < 2 * NT; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float* at = all + (row + (k >> 1) * 8) * C::ROWS + 8 * i + 2 * (w.lane & 3) + (k & 1);
          *at = g ? *at + sum[i][k] : sum[i][k];
        }
  }
  __syncthreads();
  const int high = p.source.high, wide = p.source.wide, nx = 2 * wide - 1, size = (2 * high - 1) * nx;
  for (int i = threadIdx.x; i < size; i += C::THREADS) {
    const int dy = i / nx - (high - 1), dx = i % nx - (wide - 1);
    float v = 0.f;
    for (int y = max(0, dy); y < min(high, high + dy); ++y)
      for (int x = max(0, dx); x < min(wide, wide + dx); ++x) v += all[(y * wide + x) * C::ROWS + (y - dy) * wide + x - dx];
    p.part[(static_cast<long long>(blockIdx.y) * size + i) * heads + w.head] = v;
  }
}

// Sums of the runs, in their order, eight sequences of them beside one another: out[i] (+)= sum_r part[r][i].
__global__ void __launch_bounds__(256) small_join_kernel(const float* part, float* out, int runs, int size, int add) {
  __shared__ float sums[8][32];
  chain_point();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, i = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (i < size) {
#pragma unroll 4
    for (int r = warp; r < runs; r += 8) s += part[static_cast<long long>(r) * size + i];
  }
  sums[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && i < size) {
    s = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) s += sums[k][lane];
    out[i] = add ? out[i] + s : s;
  }
}

// CTAs of a head: no more than the SMs hold of all heads at once (a few more would run behind all others: 1,000 windows of 8 x 8, 8 heads
// of 32, gradients 169 us, so 105), each with a window at least for every group.
template <int NT>
int small_runs(int n_win, int heads, int d, bool backward) {
  using C = SmallCfg<NT>;
  const int held = num_sms() * C::held(d, backward, C::stages(d, backward)) / heads, need = (n_win + C::GROUPS - 1) / C::GROUPS;
  return held < 1 ? 1 : held < need ? held : need;
}
int small_runs(int n_win, int n, int heads, int d, bool backward) {
  switch ((n + 15) / 16) {
    case 1: return small_runs<1>(n_win, heads, d, backward);
    case 2: return small_runs<2>(n_win, heads, d, backward);
    case 3: return small_runs<3>(n_win, heads, d, backward);
    case 4: return small_runs<4>(n_win, heads, d, backward);
    case 5: return small_runs<5>(n_win, heads, d, backward);
    default: return small_runs<6>(n_win, heads, d, backward);
  }
}

template <int NT>
int launch_small(SmallParams p, bool backward, cudaStream_t stream) {
  using C = SmallCfg<NT>;
  static std::atomic<uint64_t> done[2];
  p.stages = C::stages(p.d, backward);
  const int bytes = C::bytes(p.d, backward, p.stages);
  const dim3 grid(p.source.heads, p.runs);
  if (backward) {
    if (!allow_smem_once(small_bwd_kernel<NT>, SMALL_MOST, done[0])) return -20;
    return launch_chained(small_bwd_kernel<NT>, grid, C::THREADS, bytes, stream, p);
  }
  if (!allow_smem_once(small_fwd_kernel<NT>, SMALL_MOST, done[1])) return -20;
  return launch_chained(small_fwd_kernel<NT>, grid, C::THREADS, bytes, stream, p);
}
int launch_small(const SmallParams& p, bool backward, cudaStream_t stream) {
  switch ((p.n + 15) / 16) {
    case 1: return launch_small<1>(p, backward, stream);
    case 2: return launch_small<2>(p, backward, stream);
    case 3: return launch_small<3>(p, backward, stream);
    case 4: return launch_small<4>(p, backward, stream);
    case 5: return launch_small<5>(p, backward, stream);
    default: return launch_small<6>(p, backward, stream);
  }
}

}  // namespace

}  // namespace aeris
