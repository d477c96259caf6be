// Linear layers of the plain block: products with bias, activation and residual in the epilogue, and their gradients.
//
//   z = x w^T + b, y = r + act(z)
//   dz = dy act'(z), db = sum dz, dx = dz w, dw = dz^T x                                    (sums over rows)
//
// Any number of rows and columns: operand tiles that reach past a matrix are filled with zeros by the tensor maps, results
// past it are clipped by them or, where rows do not start on 16-byte boundaries or end between them, masked element by element.
// fp32 accumulation;
// bias, activation and residual are applied to the accumulators, which are rounded once.
#include "common.cuh"
#include "api.h"
#include "cluster.cuh"
#include "host.h"

namespace aeris {

namespace {

constexpr int LIN_BM = 128, LIN_BK = 64;
enum : int { LIN_OUT = 0, LIN_PART = 1 };      // bf16 results; fp32 sums of slices of the reduction

struct LinParams {
  int M, N, K, act, mode, k_splits, bias_bf16;
  __nv_bfloat16* C;
  long long ldc;
  const void* bias;
  const __nv_bfloat16* resid;
  long long ldr;
  __nv_bfloat16* Z;
  long long ldz;
  float* part;              // [k_splits, M, ld_part]
  long long ld_part;
  int c_map, z_map, r_vec;  // C, Z: rows leave as tiled stores; resid: rows of whole vectors
  int* status;
};

// exp(-z^2 / 2) and the Gaussian distribution function of z: erfc by the rational approximation in 1 / (1 + p x) times exp(-x^2)
// of Abramowitz and Stegun, 7.1.26, whose absolute error is below 1.5e-7. Next to CUDA's erff it takes half the instructions,
// shares its exponential with the derivative and does not cancel far below zero. Relative to z cdf(z) it is off by up to 5e-5 at
// z = -3, 1.6e-3 at -5, 3.6e-3 at -6 (half a step of bf16, of values of 6e-9), 1e-2 at -8; the absolute error of GELU is at most
// 2.1e-7 everywhere.
__device__ __forceinline__ void gauss(float z, float& e, float& cdf) {
  const float x = fabsf(z) * 0.70710678118654752f;
  const float t = 1.f / fmaf(0.3275911f, x, 1.f);
  e = __expf(-x * x);
  float p = fmaf(1.061405429f, t, -1.453152027f);
  p = fmaf(p, t, 1.421413741f);
  p = fmaf(p, t, -0.284496736f);
  p = fmaf(p, t, 0.254829592f);
  const float tail = 0.5f * (p * t) * e;
  cdf = z < 0.f ? tail : 1.f - tail;
}
__device__ __forceinline__ float sigmoid(float z) { return 1.f / (1.f + __expf(-z)); }

// gelu_tanh by 0.5 (1 + tanh u) = 1 / (1 + exp(-2 u)), which keeps the relative precision of small results.
__device__ __forceinline__ float act_of(float z, int act) {
  switch (act) {
    case LIN_ACT_RELU: return z < 0.f ? 0.f : z;      // a NaN stays
    case LIN_ACT_SILU: return z * sigmoid(z);
    case LIN_ACT_GELU: { float e, c; gauss(z, e, c); return z * c; }
    case LIN_ACT_GELU_TANH: return z * sigmoid(z * fmaf(z * z, 0.07135481282f, 1.59576912161f));
    default: return z;
  }
}
__device__ __forceinline__ float act_grad(float z, int act) {
  switch (act) {
    case LIN_ACT_RELU: return z > 0.f ? 1.f : 0.f;
    case LIN_ACT_SILU: { const float s = sigmoid(z); return s * fmaf(z, 1.f - s, 1.f); }
    case LIN_ACT_GELU: { float e, c; gauss(z, e, c); return fmaf(z * 0.39894228040143268f, e, c); }
    case LIN_ACT_GELU_TANH: {
      z = z > 100.f ? 100.f : z < -100.f ? -100.f : z;      // 1 and 0 long before; the square of a large one would be infinite
      const float s = sigmoid(z * fmaf(z * z, 0.07135481282f, 1.59576912161f));
      return s * fmaf(z * (1.f - s), fmaf(z * z, 3.f * 0.07135481282f, 1.59576912161f), 1.f);
    }
    default: return 1.f;
  }
}

// 32 columns from column `c` of the bias, zeros past the matrix. The same for all lanes.
__device__ __forceinline__ void bias32(const LinParams& p, int c, float (&b)[32]) {
  const bool vec = (reinterpret_cast<uintptr_t>(p.bias) & 15) == 0 && c + 32 <= p.N;
  if (!p.bias_bf16) {
    const float* s = static_cast<const float*>(p.bias) + c;
    if (vec) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float4 f = reinterpret_cast<const float4*>(s)[i];
        b[4 * i] = f.x; b[4 * i + 1] = f.y; b[4 * i + 2] = f.z; b[4 * i + 3] = f.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i) b[i] = c + i < p.N ? s[i] : 0.f;
    }
    return;
  }
  const __nv_bfloat16* s = static_cast<const __nv_bfloat16*>(p.bias) + c;
#pragma unroll
  for (int i = 0; i < 32; ++i) b[i] = c + i < p.N ? __bfloat162float(s[i]) : 0.f;
}

template <int ACT>
__device__ __forceinline__ void act32(uint32_t (&v)[32]) {
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(act_of(__uint_as_float(v[i]), ACT));
}

// bf16 columns of a warp's 32 rows on their way out, 32 at a time: two buffers each for y and z, which one lane hands to the TMA
// unit as 32 x 32 tiles (64-byte swizzle); what lies past the matrix is clipped (see lin_maps).
struct LinOut {
  uint8_t* stage;        // 8 KB: y, y, z, z of 2 KB
  int lane, n = 0;
  __device__ __forceinline__ void begin() const {       // the buffers of the step before the last one are free
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
    __syncwarp();
  }
  __device__ __forceinline__ void put(int which, const uint32_t (&o)[16]) const {
    uint8_t* b = stage + which * 4096 + (n & 1) * 2048 + lane * 64;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *reinterpret_cast<uint4*>(b + ((i ^ ((lane >> 1) & 3)) << 4)) = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
  }
  __device__ __forceinline__ void send(const CUtensorMap* my, const CUtensorMap* mz, int col, int row, int rows) {
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      if (row < rows) {
        if (my) tma_store_2d(my, stage + (n & 1) * 2048, col, row);
        if (mz) tma_store_2d(mz, stage + 4096 + (n & 1) * 2048, col, row);
      }
      asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    }
    __syncwarp();
    ++n;
  }
  __device__ __forceinline__ void drain() const {       // before the warp leaves: its copies have been performed
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
};

// 32 rows x 32 columns of a warp to rows that start anywhere, through its staging: a lane per column, so that a store is 64 bytes of
// one row (a lane per row, column by column: 1111 x 777 -> 333 15.3 us, so 8.5). `rows`, `cols`: how many there are.
__device__ __forceinline__ void store_anywhere(uint8_t* stage, int lane, const uint32_t (&o)[16], __nv_bfloat16* dst, long long ld, int rows,
                                               int cols) {
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 16; ++i) *reinterpret_cast<uint32_t*>(stage + lane * 68 + 4 * i) = o[i];       // rows of 68 bytes: 17 banks apart
  __syncwarp();
  if (lane < cols)
#pragma unroll 8
    for (int r = 0; r < rows; ++r)
      reinterpret_cast<unsigned short*>(dst)[r * ld + lane] = *reinterpret_cast<const unsigned short*>(stage + r * 68 + 2 * lane);
  __syncwarp();
}

// One thread = one accumulator row; columns [c_lo, c_hi) of the tile whose first column is col0 and lies at `taddr`.
__device__ __forceinline__ void lin_epilogue_row(const LinParams& p, uint32_t taddr, int row, bool row_ok, int col0, int c_lo,
                                                 int c_hi, int split, bool kempty, LinOut& out, const CUtensorMap* my,
                                                 const CUtensorMap* mz) {
  if (p.mode == LIN_PART) {
    float* dst = p.part + (static_cast<long long>(split) * p.M + row) * p.ld_part + col0;      // pitch a multiple of 4
#pragma unroll 1
    for (int c = c_lo; c < c_hi && col0 + c < p.N; c += 32) {
      uint32_t v[32];
      tmem_ld32(taddr + c, v);
      tmem_wait_ld();
      if (row_ok) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (col0 + c + 4 * i < p.N)
            *reinterpret_cast<float4*>(dst + c + 4 * i) =
                kempty ? make_float4(0.f, 0.f, 0.f, 0.f)
                       : make_float4(__uint_as_float(v[4 * i]), __uint_as_float(v[4 * i + 1]), __uint_as_float(v[4 * i + 2]),
                                     __uint_as_float(v[4 * i + 3]));
      }
    }
    return;
  }
  const __nv_bfloat16* res = p.resid && row_ok ? p.resid + static_cast<long long>(row) * p.ldr + col0 : nullptr;
#pragma unroll 1
  for (int c = c_lo; c < c_hi && col0 + c < p.N; c += 32) {
    uint32_t v[32], o[16];
    const int n = min(32, p.N - col0 - c);
    tmem_ld32(taddr + c, v);
    uint4 r4[4];
    const bool r_vec = res && p.r_vec && n == 32;
    if (r_vec) {
#pragma unroll
      for (int i = 0; i < 4; ++i) r4[i] = reinterpret_cast<const uint4*>(res + c)[i];
    }
    tmem_wait_ld();
    if (my || mz) out.begin();
    if (p.bias) {
      float b[32];
      bias32(p, col0 + c, b);
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) + b[i]);
    }
    if (p.Z) {
#pragma unroll
      for (int i = 0; i < 16; ++i) o[i] = pack_bf16x2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
      if (mz) out.put(1, o);
      else store_anywhere(out.stage + 4096, out.lane, o, p.Z + (row - out.lane) * p.ldz + col0 + c, p.ldz, min(32, p.M - row + out.lane), n);
    }
    switch (p.act) {
      case LIN_ACT_RELU: act32<LIN_ACT_RELU>(v); break;
      case LIN_ACT_SILU: act32<LIN_ACT_SILU>(v); break;
      case LIN_ACT_GELU: act32<LIN_ACT_GELU>(v); break;
      case LIN_ACT_GELU_TANH: act32<LIN_ACT_GELU_TANH>(v); break;
      default: break;
    }
    if (r_vec) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t w[4] = {r4[i].x, r4[i].y, r4[i].z, r4[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f = unpack_bf16x2(w[j]);
          v[8 * i + 2 * j] = __float_as_uint(__uint_as_float(v[8 * i + 2 * j]) + f.x);
          v[8 * i + 2 * j + 1] = __float_as_uint(__uint_as_float(v[8 * i + 2 * j + 1]) + f.y);
        }
      }
    } else if (res) {
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (i < n) v[i] = __float_as_uint(__uint_as_float(v[i]) + __bfloat162float(res[c + i]));
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) o[i] = pack_bf16x2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
    if (my) out.put(0, o);
    else store_anywhere(out.stage, out.lane, o, p.C + (row - out.lane) * p.ldc + col0 + c, p.ldc, min(32, p.M - row + out.lane), n);
    if (my || mz) out.send(my, mz, col0 + c, row - out.lane, p.M);
  }
}

// 128 x BN tiles, one CTA each. Warps: 0 loads, 1 issues products and owns the tensor memory, 2..5 the epilogue.
template <int BN> struct LinSmem {
  static constexpr int A_BYTES = LIN_BM * LIN_BK * 2, B_BYTES = BN * LIN_BK * 2, STAGE = A_BYTES + B_BYTES;
  static constexpr int STAGES = BN == 256 ? 4 : BN == 128 ? 5 : 7;
  static constexpr int BARS = STAGES * STAGE, OUT = BARS + 1024, TOTAL = OUT + 4 * 8192 + 1024;
  static constexpr int TMEM = 2 * BN;
  static_assert(TOTAL <= 227 * 1024, "shared memory");
};
constexpr int LIN_THREADS = 192;

// CTA `cta` of `ctas` that share a product.
template <int BN, int A_MN, int B_MN>
__device__ __forceinline__ void lin_cta(const CUtensorMap& tm_a, const CUtensorMap& tm_b, const CUtensorMap& tm_y, const CUtensorMap& tm_z,
                                        const LinParams& p, int cta, int ctas) {
  using S = LinSmem<BN>;
  static_assert(!B_MN || BN % 64 == 0, "boxes of 64 columns");
  constexpr int STAGES = S::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + S::BARS);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* tfull_bar = empty_bar + STAGES;
  uint64_t* tempty_bar = tfull_bar + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty_bar + 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  {  // an earlier kernel already failed: leave before touching TMEM (decision made once per CTA)
    __shared__ int s_abort;
    if (threadIdx.x == 0) s_abort = failed(p.status) ? 1 : 0;
    __syncthreads();
    if (s_abort) { chain_point(); return; }
  }
  const int m_tiles = (p.M + LIN_BM - 1) / LIN_BM, n_tiles = (p.N + BN - 1) / BN;
  const int kb_total = (p.K + LIN_BK - 1) / LIN_BK, kb_per_split = (kb_total + p.k_splits - 1) / p.k_splits;
  const int mn_tiles = m_tiles * n_tiles, total_tiles = mn_tiles * p.k_splits;

  if (threadIdx.x == 0) {
    prefetch_tmap(&tm_a);
    prefetch_tmap(&tm_b);
    for (int s = 0; s < STAGES; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
    for (int a = 0; a < 2; ++a) { mbar_init(&tfull_bar[a], 1); mbar_init(&tempty_bar[a], 4); }
    fence_barrier_init();
  }
  if (warp == 1) { tmem_alloc(tmem_slot, S::TMEM); tmem_relinquish(); }
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
      for (int tile = cta; tile < total_tiles && ok; tile += ctas) {
        const int split = tile / mn_tiles, mn = tile - split * mn_tiles, tm = mn / n_tiles, tn = mn - tm * n_tiles;
        const int kb0 = split * kb_per_split, kb1 = min(kb_total, kb0 + kb_per_split);
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait(&empty_bar[stage], phase ^ 1, p.status, ERR_TIMEOUT_EMPTY)) { ok = false; break; }
          uint8_t* sa = smem + stage * S::STAGE;
          uint8_t* sb = sa + S::A_BYTES;
          mbar_expect_tx(&full_bar[stage], S::STAGE);
          if constexpr (A_MN == 0) {
            tma_load_2d(sa, &tm_a, &full_bar[stage], kb * LIN_BK, tm * LIN_BM);
          } else {
#pragma unroll
            for (int j = 0; j < LIN_BM / 64; ++j)
              tma_load_2d(sa + j * 8192, &tm_a, &full_bar[stage], tm * LIN_BM + j * 64, kb * LIN_BK);
          }
          if constexpr (B_MN == 0) {
            tma_load_2d(sb, &tm_b, &full_bar[stage], kb * LIN_BK, tn * BN);
          } else {
#pragma unroll
            for (int j = 0; j < BN / 64; ++j)
              tma_load_2d(sb + j * 8192, &tm_b, &full_bar[stage], tn * BN + j * 64, kb * LIN_BK);
          }
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
      }
      if (ok)       // every stage has been released: no copy is under way at exit
        for (int s = 0; s < STAGES; ++s) {
          if (!mbar_wait(&empty_bar[stage], phase ^ 1, p.status, ERR_TIMEOUT_EMPTY)) break;
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
    }
  } else if (warp == 1) {
    if (elect_one_sync()) {
      constexpr uint32_t idesc = make_idesc_bf16(LIN_BM, BN, A_MN, B_MN);
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int tile = cta; tile < total_tiles && ok; tile += ctas) {
        const int split = tile / mn_tiles;
        const int kb0 = split * kb_per_split, kb1 = min(kb_total, kb0 + kb_per_split);
        if (!mbar_wait(&tempty_bar[acc], acc_phase ^ 1, p.status, ERR_TIMEOUT_TMEM_EMPTY)) { ok = false; break; }
        tc_fence_after();
        const uint32_t tmem_acc = tmem_base + acc * BN;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait(&full_bar[stage], phase, p.status, ERR_TIMEOUT_FULL)) { ok = false; break; }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + stage * S::STAGE), sb = sa + S::A_BYTES;
#pragma unroll
          for (int kk = 0; kk < LIN_BK / 16; ++kk) {
            const uint64_t ad = A_MN ? make_smem_desc(sa + kk * 2048, 8192, 1024) : make_smem_desc(sa + kk * 32, 0, 1024);
            const uint64_t bd = B_MN ? make_smem_desc(sb + kk * 2048, 8192, 1024) : make_smem_desc(sb + kk * 32, 0, 1024);
            umma_ss(tmem_acc, ad, bd, idesc, (kb > kb0 || kk > 0) ? 1u : 0u);
          }
          tc_commit(&empty_bar[stage]);
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
        if (!ok) break;
        tc_commit(&tfull_bar[acc]);
        if (++acc == 2) { acc = 0; acc_phase ^= 1; }
      }
    }
  } else if (warp < LIN_THREADS / 32) {
    const int q = warp & 3;  // TMEM lane quarter this warp may access
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    const bool keep = !failed(p.status);       // see note_failure
    LinOut out{smem + S::OUT + q * 8192, lane};
    for (int tile = cta; tile < total_tiles && ok; tile += ctas) {
      const int split = tile / mn_tiles, mn = tile - split * mn_tiles, tm = mn / n_tiles, tn = mn - tm * n_tiles;
      ok = __all_sync(0xffffffffu, mbar_wait(&tfull_bar[acc], acc_phase, p.status, ERR_TIMEOUT_TMEM_FULL));
      if (!ok) break;
      tc_fence_after();
      const int row = tm * LIN_BM + q * 32 + lane;
      const uint32_t taddr = tmem_base + acc * BN + (static_cast<uint32_t>(q * 32) << 16);
      if (keep)
        lin_epilogue_row(p, taddr, row, row < p.M, tn * BN, 0, BN, split, split * kb_per_split >= kb_total, out,
                         p.c_map ? &tm_y : nullptr, p.z_map ? &tm_z : nullptr);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tempty_bar[acc]);
      if (++acc == 2) { acc = 0; acc_phase ^= 1; }
    }
    out.drain();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem_base, S::TMEM);
}

template <int BN, int A_MN, int B_MN>
__global__ void __launch_bounds__(LIN_THREADS, 1)
lin_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
           const __grid_constant__ CUtensorMap tm_y, const __grid_constant__ CUtensorMap tm_z, const LinParams p) {
  lin_cta<BN, A_MN, B_MN>(tm_a, tm_b, tm_y, tm_z, p, blockIdx.x, gridDim.x);
}

// 256 x 256 tiles by CTA pairs (a cluster of two), which share the operands' reads from L2 and from shared memory: each CTA loads
// its 128 rows of A and half of B's tile, the leader issues products of both (tcgen05.mma.cta_group::2), each CTA writes its
// rows. Roles and barriers as in gemm2.cu. EW: epilogue warps, eight (two for 32 rows) for the price of one of the ring's stages
// where results leave in bf16: us, four / eight, 64800 x 1536 -> 4096 plain 543 / 522, GELU 641 / 576, with z 696 / 631, residual 739 /
// 604, 28800 x 768 -> 2048 105 / 80, 152 / 116, 162 / 122, 175 / 117. 64,800 x 1536 -> 4096 with GELU and z, 631 us, are 1.29
// PFLOP/s, of the 1.40 that a product holds under the power cap.
constexpr int LIN2_BN = 256, LIN2_STAGE = 32768;
template <int EW> struct Lin2Smem {
  static constexpr int STAGES = EW == 8 ? 5 : 6;
  static constexpr int BARS = STAGES * LIN2_STAGE, OUT = BARS + 1024, TOTAL = OUT + EW * 8192 + 1024;
  static constexpr int THREADS = 64 + 32 * EW;
  static_assert(TOTAL <= 227 * 1024, "shared memory");
};

template <int A_MN, int B_MN, int EW>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Lin2Smem<EW>::THREADS, 1)
lin2_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
            const __grid_constant__ CUtensorMap tm_y, const __grid_constant__ CUtensorMap tm_z, const LinParams p) {
  using S = Lin2Smem<EW>;
  constexpr int STAGES = S::STAGES, GROUP_M = 8;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + S::BARS);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* tfull_bar = empty_bar + STAGES;           // [2]
  uint64_t* tempty_bar = tfull_bar + 2;               // [2], in the leader: an arrival per epilogue warp of both CTAs
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty_bar + 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t crank = cluster_ctarank();
  const int cluster = blockIdx.x >> 1, n_clusters = gridDim.x >> 1;

  const int m_tiles = (p.M + 255) / 256, n_tiles = (p.N + LIN2_BN - 1) / LIN2_BN;
  const int kb_total = (p.K + LIN_BK - 1) / LIN_BK, kb_per_split = (kb_total + p.k_splits - 1) / p.k_splits;
  const int mn_tiles = m_tiles * n_tiles, total_tiles = mn_tiles * p.k_splits;
  // eight rows of tiles at a time: what the pairs at work read of A and B stays in L2
  auto tile_at = [&](int tile, int& split, int& tm, int& tn) {
    split = tile / mn_tiles;
    const int mn = tile - split * mn_tiles, g = mn / (GROUP_M * n_tiles), in = mn - g * GROUP_M * n_tiles;
    const int gm = min(GROUP_M, m_tiles - g * GROUP_M);
    tn = in / gm;
    tm = g * GROUP_M + in - tn * gm;
  };
  if (threadIdx.x == 0) {
    prefetch_tmap(&tm_a);
    prefetch_tmap(&tm_b);
    for (int s = 0; s < STAGES; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
    for (int a = 0; a < 2; ++a) { mbar_init(&tfull_bar[a], 1); mbar_init(&tempty_bar[a], 2 * EW); }
    fence_barrier_init();
  }
  if (warp == 1) { tmem_alloc2(tmem_slot, 2 * LIN2_BN); tmem_relinquish2(); }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();       // both CTAs' barriers are initialised and tensor memory is allocated before anyone signals
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  chain_point();

  if (warp == 0) {
    if (elect_one_sync()) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = cluster; tile < total_tiles && ok; tile += n_clusters) {
        int split, tm, tn;
        tile_at(tile, split, tm, tn);
        const int kb0 = split * kb_per_split, kb1 = min(kb_total, kb0 + kb_per_split), m0 = tm * 256 + crank * 128;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait_poll(&empty_bar[stage], phase ^ 1, p.status, ERR_TIMEOUT_EMPTY)) { ok = false; break; }
          uint8_t* sa = smem + stage * LIN2_STAGE;
          uint8_t* sb = sa + 16384;
          if (crank == 0) mbar_expect_tx(&full_bar[stage], 2 * LIN2_STAGE);       // both CTAs' copies
          const uint32_t fb = map_to_cta(smem_u32(&full_bar[stage]), 0);
          if constexpr (A_MN == 0) {
            tma_load_2d_pair(sa, &tm_a, fb, kb * LIN_BK, m0);
          } else {
#pragma unroll
            for (int j = 0; j < 2; ++j) tma_load_2d_pair(sa + j * 8192, &tm_a, fb, m0 + j * 64, kb * LIN_BK);
          }
          const int n0 = tn * LIN2_BN + crank * 128;
          if constexpr (B_MN == 0) {
            tma_load_2d_pair(sb, &tm_b, fb, kb * LIN_BK, n0);
          } else {
#pragma unroll
            for (int j = 0; j < 2; ++j) tma_load_2d_pair(sb + j * 8192, &tm_b, fb, n0 + j * 64, kb * LIN_BK);
          }
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
      }
      // after a time-out: the tiles that the issuer did not take, of both CTAs (a stage never filled counts as there)
      for (int s = 0; s < STAGES && !ok && crank == 0; ++s) {
        if (--stage < 0) { stage = STAGES - 1; phase ^= 1; }
        if (!mbar_wait_poll(&full_bar[stage], phase, nullptr, 0)) break;
      }
    }
  } else if (warp == 1) {
    if (crank == 0 && elect_one_sync()) {
      constexpr uint32_t idesc = make_idesc_bf16(256, LIN2_BN, A_MN, B_MN);
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int tile = cluster; tile < total_tiles && ok; tile += n_clusters) {
        const int split = tile / mn_tiles;
        const int kb0 = split * kb_per_split, kb1 = min(kb_total, kb0 + kb_per_split);
        if (!mbar_wait_poll(&tempty_bar[acc], acc_phase ^ 1, p.status, ERR_TIMEOUT_TMEM_EMPTY)) { ok = false; break; }
        tc_fence_after();
        const uint32_t tmem_acc = tmem_base + acc * LIN2_BN;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait_poll(&full_bar[stage], phase, p.status, ERR_TIMEOUT_FULL)) { ok = false; break; }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + stage * LIN2_STAGE), sb = sa + 16384;
#pragma unroll
          for (int kk = 0; kk < LIN_BK / 16; ++kk) {
            const uint64_t ad = A_MN ? make_smem_desc(sa + kk * 2048, 8192, 1024) : make_smem_desc(sa + kk * 32, 0, 1024);
            const uint64_t bd = B_MN ? make_smem_desc(sb + kk * 2048, 8192, 1024) : make_smem_desc(sb + kk * 32, 0, 1024);
            umma2_ss(tmem_acc, ad, bd, idesc, (kb > kb0 || kk > 0) ? 1u : 0u);
          }
          tc_commit2_mc(&empty_bar[stage], 0x3);
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
        if (!ok) break;
        tc_commit2_mc(&tfull_bar[acc], 0x3);
        if (++acc == 2) { acc = 0; acc_phase ^= 1; }
      }
      // the last products have completed: an epilogue that gave up has not waited for them
      if (--stage < 0) { stage = STAGES - 1; phase ^= 1; }
      mbar_wait_poll(&empty_bar[stage], phase, nullptr, 0);
    }
  } else {
    const int q = warp & 3, part = (warp - 2) >> 2;
    int acc = 0;
    uint32_t acc_phase = 0;
    const bool keep = !failed(p.status);       // see note_failure
    const uint32_t leader_tempty = map_to_cta(smem_u32(&tempty_bar[0]), 0);
    LinOut out{smem + S::OUT + (part * 4 + q) * 8192, lane};
    for (int tile = cluster; tile < total_tiles; tile += n_clusters) {
      int split, tm, tn;
      tile_at(tile, split, tm, tn);
      if (!__all_sync(0xffffffffu, mbar_wait_poll(&tfull_bar[acc], acc_phase, p.status, ERR_TIMEOUT_TMEM_FULL))) break;
      tc_fence_after();
      const int row = tm * 256 + crank * 128 + q * 32 + lane;
      const uint32_t taddr = tmem_base + acc * LIN2_BN + (static_cast<uint32_t>(q * 32) << 16);
      constexpr int COLS = LIN2_BN / (EW / 4);
      if (keep)
        lin_epilogue_row(p, taddr, row, row < p.M, tn * LIN2_BN, part * COLS, (part + 1) * COLS, split,
                         split * kb_per_split >= kb_total, out, p.c_map ? &tm_y : nullptr, p.z_map ? &tm_z : nullptr);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_remote(leader_tempty + acc * 8);
      if (++acc == 2) { acc = 0; acc_phase ^= 1; }
    }
    out.drain();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();       // nobody leaves while the pair may still touch its shared memory or tensor memory
  tc_fence_after();
  if (warp == 1) tmem_dealloc2(tmem_base, 2 * LIN2_BN);
}

bool whole_rows(const void* base, long long ld) { return (reinterpret_cast<uintptr_t>(base) & 15) == 0 && ld % 8 == 0; }

struct LinMaps {
  CUtensorMap a, b, y, z;
};
// Tensor maps of a product whose tiles take `rows_a` rows of A and `rows_b` of B at a time; decides how results leave.
template <int A_MN, int B_MN>
int lin_maps(LinMaps& m, const void* A, long long lda, const void* B, long long ldb, LinParams& p, int rows_a, int rows_b) {
  int r;
  if (!whole_rows(A, lda) || !whole_rows(B, ldb)) return -11;
  if ((r = A_MN ? make_tmap_2d_bf16(&m.a, A, p.M, p.K, lda, 64, LIN_BK) : make_tmap_2d_bf16(&m.a, A, p.K, p.M, lda, LIN_BK, rows_a)))
    return r;
  if ((r = B_MN ? make_tmap_2d_bf16(&m.b, B, p.N, p.K, ldb, 64, LIN_BK) : make_tmap_2d_bf16(&m.b, B, p.K, p.N, ldb, LIN_BK, rows_b)))
    return r - 100;
  m.y = m.z = m.a;         // not stored through where rows go element by element
  // A tiled store clips columns in pieces of 16 bytes: it would write zeros behind a row that ends inside one (28,800 x 768 -> 2047
  // into rows of 2048, GELU: 96 us with it, 130 without, and with z 107 and 176)
  const bool pieces = p.mode == LIN_OUT && p.N % 8 == 0;
  p.c_map = pieces && whole_rows(p.C, p.ldc);
  p.z_map = pieces && p.Z && whole_rows(p.Z, p.ldz);
  p.r_vec = p.resid && whole_rows(p.resid, p.ldr);
  if (p.c_map && (r = make_tmap_2d_sw64_bf16(&m.y, p.C, p.N, p.M, p.ldc, 32, 32))) return r - 200;
  if (p.z_map && (r = make_tmap_2d_sw64_bf16(&m.z, p.Z, p.N, p.M, p.ldz, 32, 32))) return r - 300;
  return 0;
}

long long lin_tiles(int M, int N, int bm, int bn) { return static_cast<long long>((M + bm - 1) / bm) * ((N + bn - 1) / bn); }

template <int BN, int A_MN, int B_MN>
int launch_lin(const void* A, long long lda, const void* B, long long ldb, LinParams p, cudaStream_t stream) {
  using S = LinSmem<BN>;
  auto kern = lin_kernel<BN, A_MN, B_MN>;
  static std::atomic<uint64_t> done{0};
  if (!allow_smem_once(kern, S::TOTAL, done)) return -20;
  LinMaps m;
  const int r = lin_maps<A_MN, B_MN>(m, A, lda, B, ldb, p, LIN_BM, BN);
  if (r) return r;
  const long long tiles = lin_tiles(p.M, p.N, LIN_BM, BN) * p.k_splits;
  if (tiles > 0x3fffffff) return -2;
  const int grid = tiles < num_sms() ? static_cast<int>(tiles) : num_sms();
  return launch_chained(kern, grid, LIN_THREADS, S::TOTAL, stream, m.a, m.b, m.y, m.z, p);
}

template <int A_MN, int B_MN, int EW>
int launch_lin2(const void* A, long long lda, const void* B, long long ldb, LinParams p, cudaStream_t stream) {
  using S = Lin2Smem<EW>;
  auto kern = lin2_kernel<A_MN, B_MN, EW>;
  static std::atomic<uint64_t> done{0};
  if (!allow_smem_once(kern, S::TOTAL, done)) return -20;
  LinMaps m;
  const int r = lin_maps<A_MN, B_MN>(m, A, lda, B, ldb, p, 128, 128);
  if (r) return r;
  const long long tiles = lin_tiles(p.M, p.N, 256, LIN2_BN) * p.k_splits;
  if (tiles > 0x1fffffff) return -2;
  // as many pairs as the device holds at once (a group of SMs with an odd number of them has one left over)
  static std::atomic<int> held{0};
  int pairs = held.load(std::memory_order_relaxed);
  if (!pairs) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(num_sms() / 2 * 2);
    cfg.blockDim = dim3(S::THREADS);
    cfg.dynamicSmemBytes = S::TOTAL;
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim = {2, 1, 1};
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&pairs, kern, &cfg) != cudaSuccess || pairs <= 0) pairs = num_sms() / 2;
    held.store(pairs, std::memory_order_relaxed);
  }
  const int clusters = tiles < pairs ? static_cast<int>(tiles) : pairs;
  return launch_chained(kern, 2 * clusters, S::THREADS, S::TOTAL, stream, m.a, m.b, m.y, m.z, p);
}

// Few rows: a warp per two columns, whose weights it reads once while x lies in shared memory. The tensor core's tiles are 128 rows
// high whatever there is of them; one row of 1536 -> 4096 takes them 9.7 us, this kernel 3.6, which is the weights' way from L2 (3.5 TB/s).
constexpr int ROWS_MAX = 8, ROWS_COLS = 2, ROWS_WARPS = 8;
template <int M>
__global__ void __launch_bounds__(32 * ROWS_WARPS) lin_rows_kernel(const LinParams p, const __nv_bfloat16* x, long long lda,
                                                                   const __nv_bfloat16* w, long long ldb) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  uint4* sx = reinterpret_cast<uint4*>(smem_raw);       // [M][vecs], zeros behind the row's end
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, vecs = (p.K + 7) / 8, whole = p.K / 8;
  chain_point();
  const int col0 = (blockIdx.x * ROWS_WARPS + warp) * ROWS_COLS;
  auto vec_of = [&](const __nv_bfloat16* row, int v) -> uint4 {
    if (v < whole) return reinterpret_cast<const uint4*>(row)[v];
    unsigned short e[8] = {};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (8 * v + i < p.K) e[i] = reinterpret_cast<const unsigned short*>(row)[8 * v + i];
    return make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
  };
  for (int i = threadIdx.x; i < M * vecs; i += 32 * ROWS_WARPS) {
    const int m = i / vecs;
    sx[i] = vec_of(x + m * lda, i - m * vecs);
  }
  __syncthreads();
  if (col0 >= p.N) return;
  const __nv_bfloat16* w0 = w + col0 * ldb;
  const __nv_bfloat16* w1 = w + min(col0 + 1, p.N - 1) * ldb;
  uint64_t acc[M][ROWS_COLS];
#pragma unroll
  for (int m = 0; m < M; ++m) acc[m][0] = acc[m][1] = 0ull;
#pragma unroll 4
  for (int v = lane; v < vecs; v += 32) {
    const uint4 a = vec_of(w0, v), b = vec_of(w1, v);
    const uint64_t fa[4] = {f2_from_bf16x2(a.x), f2_from_bf16x2(a.y), f2_from_bf16x2(a.z), f2_from_bf16x2(a.w)};
    const uint64_t fb[4] = {f2_from_bf16x2(b.x), f2_from_bf16x2(b.y), f2_from_bf16x2(b.z), f2_from_bf16x2(b.w)};
#pragma unroll
    for (int m = 0; m < M; ++m) {
      const uint4 c = sx[m * vecs + v];
      const uint64_t fx[4] = {f2_from_bf16x2(c.x), f2_from_bf16x2(c.y), f2_from_bf16x2(c.z), f2_from_bf16x2(c.w)};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        acc[m][0] = f2_fma(fx[i], fa[i], acc[m][0]);
        acc[m][1] = f2_fma(fx[i], fb[i], acc[m][1]);
      }
    }
  }
  float mine = 0.f;         // lane 2 m + c: row m, column c
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int c = 0; c < ROWS_COLS; ++c) {
      float lo, hi;
      f2_unpack(acc[m][c], lo, hi);
      float s = lo + hi;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      if (lane == 2 * m + c) mine = s;
    }
  const int m = lane >> 1, col = col0 + (lane & 1);
  if (m >= M || col >= p.N) return;
  if (p.bias)
    mine += p.bias_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p.bias)[col]) : static_cast<const float*>(p.bias)[col];
  if (p.Z) p.Z[m * p.ldz + col] = __float2bfloat16_rn(mine);
  float v = act_of(mine, p.act);
  if (p.resid) v += __bfloat162float(p.resid[m * p.ldr + col]);
  p.C[m * p.ldc + col] = __float2bfloat16_rn(v);
}

template <int M = 1>
int launch_rows(const LinParams& p, const void* x, long long ldx, const void* w, long long ldw, cudaStream_t stream) {
  if constexpr (M < ROWS_MAX) {
    if (p.M > M) return launch_rows<M + 1>(p, x, ldx, w, ldw, stream);
  }
  const int per = ROWS_WARPS * ROWS_COLS;
  return launch_chained(lin_rows_kernel<M>, (p.N + per - 1) / per, 32 * ROWS_WARPS, M * ((p.K + 7) / 8) * 16, stream, p,
                        static_cast<const __nv_bfloat16*>(x), ldx, static_cast<const __nv_bfloat16*>(w), ldw);
}

// Which kernel takes a product: the one whose rounds of tiles are over first by the cycles that a block of 64 of the reduction
// takes (fitted to what they measured, us, CTA pairs / single CTAs 256 / 128 / 64 / 32 wide, forward: 64 x 1536 -> 4096 14.8 / 14.2 /
// 9.2 / 7.4 / 6.9, 900 x 768 -> 768 10.0 / 11.3 / 7.4 / 5.8 / 6.8, 3600 x 512 -> 512 9.2 / 10.3 / 7.0 / 7.1 / 8.5, 12150 x 1152 ->
// 1152 34.3 / 34.3 / 30.3 / 40.4 / 69.5, 28800 x 768 -> 2048 76 / 85 / 90 / 112 / 196, 64800 x 1536 -> 1536 213 / 235 / 269 / 374 /
// 691; of these the rule loses 13 % at 12150 x 1152 and nothing elsewhere).
constexpr int LIN_PAIR = 0;
long long lin_cost(const LinParams& p, int bn, int splits) {
  const int kb = (p.K + LIN_BK - 1) / LIN_BK, units = bn == LIN_PAIR ? num_sms() / 2 : num_sms();
  const long long tiles = (bn == LIN_PAIR ? lin_tiles(p.M, p.N, 256, 256) : lin_tiles(p.M, p.N, 128, bn)) * splits;
  const int per = bn == LIN_PAIR ? 530 : bn == 256 ? 640 : bn == 128 ? 400 : bn == 64 ? 260 : 230;
  return (tiles + units - 1) / units * ((kb + splits - 1) / splits) * per + 4000;
}

template <int A_MN, int B_MN>
int launch_product(const void* A, long long lda, const void* B, long long ldb, const LinParams& p, cudaStream_t stream) {
  int best = LIN_PAIR;
  for (int bn : {256, 128, 64, 32})
    if ((bn > 32 || !B_MN) && lin_cost(p, bn, p.k_splits) < lin_cost(p, best, p.k_splits)) best = bn;
  switch (best) {
    case 256: return launch_lin<256, A_MN, B_MN>(A, lda, B, ldb, p, stream);
    case 128: return launch_lin<128, A_MN, B_MN>(A, lda, B, ldb, p, stream);
    case 64: return launch_lin<64, A_MN, B_MN>(A, lda, B, ldb, p, stream);
    case 32:
      if constexpr (!B_MN) return launch_lin<32, A_MN, B_MN>(A, lda, B, ldb, p, stream);
      break;
    default: break;
  }
  // dw over few rows is its results' way out (eight epilogue warps: 64 x 1536 -> 4096 11 us, four 17), over many the ring's
  if constexpr (A_MN) {
    if (p.K > 16 * LIN_BK * p.k_splits) return launch_lin2<A_MN, B_MN, 4>(A, lda, B, ldb, p, stream);
  }
  return launch_lin2<A_MN, B_MN, 8>(A, lda, B, ldb, p, stream);
}

// ------------------------------------------------------------------------------------------------ gradients' own passes
constexpr int DZ_THREADS = 256, DZ_COLS = 64;

__device__ __forceinline__ float bf(unsigned short u) { return __uint_as_float(static_cast<uint32_t>(u) << 16); }

struct DzParams {
  const void *dy, *z;
  void* dz;
  float* sums;              // [gridDim.y, cols], or null
  int add;                  // one slice: whether sums is added to
  long long ld_dy, ld_z, ld_dz;
  int rows, cols;
};
// dz = dy act'(z) and the column sums of one slice of the rows. dz is rounded to bf16, half a step of it at most (2^-8), for the tensor
// core multiplies bf16 by bf16 and the other operands are bf16: dx and dw end 2.3e-3 off where fp32 products of an unrounded dz end
// 1.7e-3 off, which is their own rounding. The sums are of the fp32 values. A thread takes V columns (one 16-byte vector, or one column
// where rows start anywhere) of every R-th row of its slice; a block 64 columns. 28,800 x 2048, GELU by tanh: 73 us, 4.9 TB/s, with
// half as many slices 78; four rows at a time and two blocks an SM 85, one row and five 92; column sums alone 24 (4.8 TB/s).
template <int V> constexpr int DZ_ROWS = DZ_THREADS / (DZ_COLS / V);
template <int V, int ACT>
__device__ __forceinline__ void dz_block(const DzParams& a, int block, int slice, int slices, float (*part)[DZ_COLS]) {
  constexpr int CT = DZ_COLS / V, R = DZ_ROWS<V>, U = ACT == LIN_ACT_NONE ? 1 : 2;     // rows asked for at a time
  const int c0 = threadIdx.x % CT * V, col = block * DZ_COLS + c0, r0 = threadIdx.x / CT;
  float s[V] = {};
  if (col < a.cols) {
    const long long step = static_cast<long long>(slices) * R;
    for (long long row = static_cast<long long>(slice) * R + r0; row < a.rows; row += U * step) {
      unsigned short d[U][V], z[U][V];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (row + u * step < a.rows) {
          const unsigned short* pd = static_cast<const unsigned short*>(a.dy) + (row + u * step) * a.ld_dy + col;
          const unsigned short* pz = static_cast<const unsigned short*>(a.z) + (row + u * step) * a.ld_z + col;
          if constexpr (V == 8) {
            *reinterpret_cast<uint4*>(d[u]) = *reinterpret_cast<const uint4*>(pd);
            if (ACT != LIN_ACT_NONE) *reinterpret_cast<uint4*>(z[u]) = *reinterpret_cast<const uint4*>(pz);
          } else {
            d[u][0] = *pd;
            if (ACT != LIN_ACT_NONE) z[u][0] = *pz;
          }
        }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (row + u * step < a.rows) {
          float g[V];
#pragma unroll
          for (int i = 0; i < V; ++i) {
            // a product by itself, so that the sums are the same bits whether dz is written or not
            g[i] = ACT != LIN_ACT_NONE ? __fmul_rn(bf(d[u][i]), act_grad(bf(z[u][i]), ACT)) : bf(d[u][i]);
            s[i] += g[i];
          }
          if (a.dz) {
            __nv_bfloat16* dz = static_cast<__nv_bfloat16*>(a.dz) + (row + u * step) * a.ld_dz + col;
            if constexpr (V == 8)
              *reinterpret_cast<uint4*>(dz) = make_uint4(pack_bf16x2(g[0], g[1]), pack_bf16x2(g[2], g[3]), pack_bf16x2(g[4], g[5]),
                                                         pack_bf16x2(g[6], g[7]));
            else
              *dz = __float2bfloat16_rn(g[0]);
          }
        }
    }
  }
  if (!a.sums) return;
#pragma unroll
  for (int i = 0; i < V; ++i) part[r0][c0 + i] = s[i];
  __syncthreads();
  const int c = block * DZ_COLS + static_cast<int>(threadIdx.x);
  if (threadIdx.x < DZ_COLS && c < a.cols) {
    float t = 0.f;
    for (int r = 0; r < R; ++r) t += part[r][threadIdx.x];
    float* out = a.sums + static_cast<long long>(slice) * a.cols + c;
    *out = a.add ? *out + t : t;
  }
}
template <int V, int ACT>
__global__ void __launch_bounds__(DZ_THREADS, ACT == LIN_ACT_NONE ? 5 : 3) lin_dz_kernel(const DzParams a) {
  __shared__ float part[DZ_ROWS<V>][DZ_COLS];
  chain_point();
  dz_block<V, ACT>(a, blockIdx.x, blockIdx.y, gridDim.y, part);
}

template <int V>
int launch_dz(const DzParams& a, int act, dim3 grid, cudaStream_t stream) {
  switch (act) {
    case LIN_ACT_RELU: return launch_chained(lin_dz_kernel<V, LIN_ACT_RELU>, grid, DZ_THREADS, 0, stream, a);
    case LIN_ACT_SILU: return launch_chained(lin_dz_kernel<V, LIN_ACT_SILU>, grid, DZ_THREADS, 0, stream, a);
    case LIN_ACT_GELU: return launch_chained(lin_dz_kernel<V, LIN_ACT_GELU>, grid, DZ_THREADS, 0, stream, a);
    case LIN_ACT_GELU_TANH: return launch_chained(lin_dz_kernel<V, LIN_ACT_GELU_TANH>, grid, DZ_THREADS, 0, stream, a);
    default: return launch_chained(lin_dz_kernel<V, LIN_ACT_NONE>, grid, DZ_THREADS, 0, stream, a);
  }
}

// Both products of the gradients in one launch, where their tiles fit beside one another: the first `n_dx` CTAs make dx, the next `n_dw`
// dw, and without an activation the last ones the bias's gradient, 64 columns each. 14 x 960 -> 64 in one launch for three: 15.4 us a
// call for 20.0, in a graph 3.9 for 8.2; 200 x 512 -> 512 with GELU 19.9 for 22.4 and 8.8 for 12.5.
struct LinBoth {
  LinMaps dx, dw;
  LinParams px, pw;
  DzParams d;
  int n_dx, n_dw, d_vec;
};
template <int BN>
__global__ void __launch_bounds__(DZ_THREADS, 1) lin_both_kernel(const __grid_constant__ LinBoth a) {
  extern __shared__ uint8_t smem_raw[];
  const int b = blockIdx.x;
  if (b < a.n_dx) {
    lin_cta<BN, 0, 1>(a.dx.a, a.dx.b, a.dx.y, a.dx.z, a.px, b, a.n_dx);
  } else if (b < a.n_dx + a.n_dw) {
    lin_cta<BN, 1, 1>(a.dw.a, a.dw.b, a.dw.y, a.dw.z, a.pw, b - a.n_dx, a.n_dw);
  } else {
    chain_point();
    float(*part)[DZ_COLS] = reinterpret_cast<float(*)[DZ_COLS]>(smem_raw);
    if (a.d_vec) dz_block<8, LIN_ACT_NONE>(a.d, b - a.n_dx - a.n_dw, 0, 1, part);
    else dz_block<1, LIN_ACT_NONE>(a.d, b - a.n_dx - a.n_dw, 0, 1, part);
  }
}

struct Operand {
  const void* p;
  long long ld;
};
template <int BN>
int launch_both(const Operand& dz, const Operand& w, const Operand& x, LinBoth& a, int n_db, cudaStream_t stream) {
  using S = LinSmem<BN>;
  static std::atomic<uint64_t> done{0};
  if (!allow_smem_once(lin_both_kernel<BN>, S::TOTAL, done)) return -20;
  int r;
  if ((r = lin_maps<0, 1>(a.dx, dz.p, dz.ld, w.p, w.ld, a.px, LIN_BM, BN))) return r;
  if ((r = lin_maps<1, 1>(a.dw, dz.p, dz.ld, x.p, x.ld, a.pw, LIN_BM, BN))) return r - 1000;
  a.n_dx = static_cast<int>(lin_tiles(a.px.M, a.px.N, LIN_BM, BN) * a.px.k_splits);
  a.n_dw = static_cast<int>(lin_tiles(a.pw.M, a.pw.N, LIN_BM, BN) * a.pw.k_splits);
  return launch_chained(lin_both_kernel<BN>, a.n_dx + a.n_dw + n_db, DZ_THREADS, S::TOTAL, stream, a);
}
// The width of the tiles with which both products go into one launch, or 0: their tiles are to fit beside one another, and the longer
// one is to be over before two launches would be.
int both_width(const LinParams& px, const LinParams& pw) {
  long long apart = 0;
  for (const LinParams* p : {&px, &pw}) {
    long long best = lin_cost(*p, LIN_PAIR, p->k_splits);
    for (int bn : {256, 128, 64}) {
      const long long c = lin_cost(*p, bn, p->k_splits);
      best = c < best ? c : best;
    }
    apart += best;
  }
  for (int bn : {64, 128}) {
    const long long tiles = lin_tiles(px.M, px.N, LIN_BM, bn) * px.k_splits + lin_tiles(pw.M, pw.N, LIN_BM, bn) * pw.k_splits;
    const long long cx = lin_cost(px, bn, px.k_splits), cw = lin_cost(pw, bn, pw.k_splits);
    if (tiles <= num_sms() && (cx > cw ? cx : cw) < apart) return bn;
  }
  return 0;
}

// Rows that start on 16-byte boundaries, for tiled loads: dst [rows, (cols + 7) / 8 * 8] of src, zeros behind the rows' ends. One or two
// matrices a launch.
struct PadJob {
  const unsigned short* src;
  uint4* dst;
  long long ld;
  int rows, cols;
};
struct PadJobs {
  PadJob job[2];
};
__global__ void __launch_bounds__(DZ_THREADS) lin_pad_kernel(const PadJobs jobs) {
  chain_point();
  const PadJob j = jobs.job[blockIdx.y];
  const int vecs = (j.cols + 7) / 8;
  const long long n = static_cast<long long>(j.rows) * vecs;
  for (long long i = static_cast<long long>(blockIdx.x) * DZ_THREADS + threadIdx.x; i < n; i += static_cast<long long>(gridDim.x) * DZ_THREADS) {
    const long long row = i / vecs;
    const int c = static_cast<int>(i - row * vecs) * 8;
    const unsigned short* s = j.src + row * j.ld + c;
    unsigned short e[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) e[k] = c + k < j.cols ? s[k] : static_cast<unsigned short>(0);
    j.dst[i] = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
  }
}

// Small layers without the tensor core, any pitch, in one launch: G neighbouring lanes per result, which share its sum. The
// gradients make dz anew for every result that needs it.
constexpr long long SMALL_FWD = 1 << 23, SMALL_BWD = 1 << 18;       // rows x inner x columns, see small_fwd and small_bwd

template <typename F>
__device__ __forceinline__ float group_sum(int n, int g, int lane, F&& term) {
  float s = 0.f;
#pragma unroll 8
  for (int k = lane; k < n; k += g) s += term(k);
  for (int o = g >> 1; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}

__global__ void __launch_bounds__(DZ_THREADS) lin_small_fwd_kernel(const LinParams p, const unsigned short* x, long long ldx,
                                                                   const unsigned short* w, long long ldw, int g) {
  chain_point();
  const long long n = static_cast<long long>(p.M) * p.N;
  const int lane = threadIdx.x % g, per = DZ_THREADS / g;
  for (long long base = static_cast<long long>(blockIdx.x) * per; base < n; base += static_cast<long long>(gridDim.x) * per) {
    const long long i = base + threadIdx.x / g, j = i < n ? i : n - 1;      // lanes of results that there are not stay for the sums
    const int row = static_cast<int>(j / p.N), col = static_cast<int>(j - static_cast<long long>(row) * p.N);
    const unsigned short *px = x + row * ldx, *pw = w + col * ldw;
    float z = group_sum(p.K, g, lane, [&](int k) { return bf(px[k]) * bf(pw[k]); });
    if (lane || i >= n) continue;
    if (p.bias)
      z += p.bias_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p.bias)[col]) : static_cast<const float*>(p.bias)[col];
    if (p.Z) p.Z[row * p.ldz + col] = __float2bfloat16_rn(z);
    float v = act_of(z, p.act);
    if (p.resid) v += __bfloat162float(p.resid[row * p.ldr + col]);
    p.C[row * p.ldc + col] = __float2bfloat16_rn(v);
  }
}

__global__ void __launch_bounds__(DZ_THREADS) lin_small_bwd_kernel(const AerisLinearGrad a, int g) {
  chain_point();
  const unsigned short *dy = static_cast<const unsigned short*>(a.dy), *zz = static_cast<const unsigned short*>(a.z),
                       *x = static_cast<const unsigned short*>(a.x), *w = static_cast<const unsigned short*>(a.w);
  auto dz = [&](int r, int c) {
    const float d = bf(dy[r * a.ld_dy + c]);
    return zz ? d * act_grad(bf(zz[r * a.ld_z + c]), a.act) : d;
  };
  const long long n_dx = a.dx ? static_cast<long long>(a.rows) * a.inner : 0, n_dw = a.dw ? static_cast<long long>(a.cols) * a.inner : 0;
  const long long n = n_dx + n_dw + (a.db ? a.cols : 0);
  const int lane = threadIdx.x % g, per = DZ_THREADS / g;
  for (long long base = static_cast<long long>(blockIdx.x) * per; base < n; base += static_cast<long long>(gridDim.x) * per) {
    long long i = base + threadIdx.x / g;
    const bool live = i < n && lane == 0;
    // a warp's lanes may be at results of two kinds: each group loops by itself, all of them meet at the sums
    float s = 0.f;
    if (i < n_dx) {
      const int r = static_cast<int>(i / a.inner), k = static_cast<int>(i - static_cast<long long>(r) * a.inner);
      for (int c = lane; c < a.cols; c += g) s = fmaf(dz(r, c), bf(w[c * a.ld_w + k]), s);
    } else if (i < n_dx + n_dw) {
      const int c = static_cast<int>((i - n_dx) / a.inner), k = static_cast<int>(i - n_dx - static_cast<long long>(c) * a.inner);
      for (int r = lane; r < a.rows; r += g) s = fmaf(dz(r, c), bf(x[r * a.ld_x + k]), s);
    } else if (i < n) {
      for (int r = lane; r < a.rows; r += g) s += dz(r, static_cast<int>(i - n_dx - n_dw));
    }
    __syncwarp();
    for (int o = g >> 1; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (!live) continue;
    if (i < n_dx) {
      const long long r = i / a.inner;
      static_cast<__nv_bfloat16*>(a.dx)[r * a.ld_dx + i - r * a.inner] = __float2bfloat16_rn(s);
    } else if (i < n_dx + n_dw) {
      i -= n_dx;
      const long long c = i / a.inner, at = c * a.ld_dw + i - c * a.inner;
      if (a.dw_f32) static_cast<float*>(a.dw)[at] += s;
      else static_cast<__nv_bfloat16*>(a.dw)[at] = __float2bfloat16_rn(s);
    } else {
      float* out = a.db + i - n_dx - n_dw;
      *out = a.add_db ? *out + s : s;
    }
  }
}

// Sums of the slices, in their order: out[c] (+)= sum_s work[s][c].
__global__ void __launch_bounds__(DZ_THREADS) lin_join_sums_kernel(const float* work, float* out, int slices, int cols, int add) {
  __shared__ float part[8][32];
  chain_point();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (c < cols)
    for (int i = warp; i < slices; i += 8) s += work[static_cast<long long>(i) * cols + c];
  part[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && c < cols) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += part[i][lane];
    out[c] = add ? out[c] + s : s;
  }
}

// dw or dx from the sums of slices of the reduction, in their order. `part`: [slices, rows, ld] fp32, ld a multiple of 4.
__global__ void __launch_bounds__(DZ_THREADS) lin_join_kernel(const float* part, void* dw, long long ld_dw, int f32, int vec,
                                                                 int slices, int rows, int cols, long long ld) {
  chain_point();
  const int per_row = (cols + 3) / 4;
  const long long n = static_cast<long long>(rows) * per_row, size = static_cast<long long>(rows) * ld;
  for (long long i = static_cast<long long>(blockIdx.x) * DZ_THREADS + threadIdx.x; i < n; i += static_cast<long long>(gridDim.x) * DZ_THREADS) {
    const long long row = i / per_row;
    const int c = static_cast<int>(i - row * per_row) * 4;
    const float* src = part + row * ld + c;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < slices; ++k) {
      const float4 v = *reinterpret_cast<const float4*>(src + k * size);
      s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
    const float v[4] = {s.x, s.y, s.z, s.w};
    if (f32) {
      float* dst = static_cast<float*>(dw) + row * ld_dw + c;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c + j < cols) dst[j] += v[j];
    } else {
      __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(dw) + row * ld_dw + c;
      if (vec && c + 4 <= cols) {
        *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (c + j < cols) dst[j] = __float2bfloat16_rn(v[j]);
      }
    }
  }
}

// Slices of the reduction over the rows of dw, of which each costs its start and its sums' way through memory as well; at most 8192
// rows a slice, for the tensor core truncates at every addition and the error of a sum grows with its length (9e-10 of it per
// row).
int slices_of(int M, int N, int K, int least) {
  LinParams p{};
  p.M = M; p.N = N; p.K = K;
  const int kb = (K + LIN_BK - 1) / LIN_BK;
  const double sums = 8.0 * M * N / 3000;      // cycles to write and read one slice's, 3 KB a cycle
  int best = least;
  double cost = 1e30;
  for (int s = least; s <= 64 && (s == least || kb / s >= 4); ++s)
    for (int bn : {LIN_PAIR, 256, 128, 64}) {
      const double c = static_cast<double>(lin_cost(p, bn, s)) + (s > 1 ? s * sums + 4000 : 0);
      if (c < cost) { cost = c; best = s; }
    }
  return best;
}
int dw_slices(int rows, int inner, int cols) { return slices_of(cols, inner, rows, (rows + 128 * LIN_BK - 1) / (128 * LIN_BK)); }
// Slices of the columns for dx, whose tiles are few where rows are: product and join of 64 x 1536 -> 4096 8 us for 14, of 5 x 2048 -> 4096
// 11 for 19. With the epilogue warps above both gradients take 19.0 us in a graph for 26.7, and 22.2 for 28.4.
int dx_slices(int rows, int inner, int cols) { return slices_of(rows, inner, cols, 1); }

}  // namespace

}  // namespace aeris

using namespace aeris;

namespace {

long long up(long long bytes) { return (bytes + 255) / 256 * 256; }
long long padded(int cols) { return (static_cast<long long>(cols) + 7) / 8 * 8; }
// A single row has no pitch of its own: one that tensor maps take.
long long pitch(long long ld, int rows, int cols) { return rows == 1 ? padded(cols) : ld; }
int blocks_for(long long threads) {
  const long long b = (threads + DZ_THREADS - 1) / DZ_THREADS, most = 16ll * num_sms();
  return static_cast<int>(b < most ? b : most);
}
// Whether tiled loads take the rows where they are.
bool tiled(const void* p, long long ld, int rows, int cols) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (rows == 1 || (ld % 8 == 0 && ld >= cols));
}
// Operands of products: where they are, or copies in the workspace, which go on behind one another and are made in one launch.
struct Operands {
  uint8_t* work;
  long long at = 0;
  PadJobs jobs{};
  int n = 0;
  long long most = 0;

  Operand add(const void* p, long long ld, int rows, int cols) {
    if (tiled(p, ld, rows, cols)) return {p, pitch(ld, rows, cols)};
    uint8_t* copy = work + at;
    at += up(2 * padded(cols) * rows);
    jobs.job[n++] = {static_cast<const unsigned short*>(p), reinterpret_cast<uint4*>(copy), ld, rows, cols};
    const long long vecs = padded(cols) / 8 * rows;
    most = most > vecs ? most : vecs;
    return {copy, padded(cols)};
  }
  int launch(int& kernels, cudaStream_t stream) {
    if (!n) return 0;
    ++kernels;
    return launch_chained(lin_pad_kernel, dim3(blocks_for(most), n), DZ_THREADS, 0, stream, jobs);
  }
};

// Slices of the rows whose column sums are taken apart: about sixteen blocks of 64 columns on every multiprocessor.
int db_slices(int rows, int cols) {
  if (rows <= (cols % 8 ? 32 : 256)) return 1;        // over before a second launch would begin
  const long long most = 16ll * num_sms() * DZ_COLS / cols + 1, need = (rows + 31ll) / 32;
  return static_cast<int>(most < need ? (most < 4096 ? most : 4096) : (need < 4096 ? need : 4096));
}
// fp32 sums of s slices; one slice of bf16 results goes straight to its place.
long long part_bytes(int s, int rows, int inner, bool f32) { return s > 1 || f32 ? up(4ll * s * rows * ((inner + 3) / 4 * 4)) : 0; }

}  // namespace

namespace {

// Whether a layer goes without the tensor core: forward where operands would have to be copied first, backward where five launches
// would cost more than the work. us a call, before / so: forward 10 x 3685 -> 100 17.9 / 13.4, backward 369 x 4 -> 2 27.5 / 14.5.
bool small_fwd(int rows, int inner, int cols, bool pad) {
  return pad && static_cast<double>(rows) * inner * cols <= SMALL_FWD;
}
bool small_bwd(int rows, int inner, int cols) { return static_cast<double>(rows) * inner * cols <= SMALL_BWD; }
// Lanes that share a sum of n terms: four terms each at least, at most a warp.
int lanes_for(int n) {
  int g = 1;
  while (g < 32 && 8 * g <= n) g *= 2;
  return g;
}

}  // namespace

extern "C" long long aeris_linear_fwd_bytes(int rows, int inner, int cols, int pad_x, int pad_w) {
  if (rows <= 0 || inner <= 0 || cols <= 0) return -1;
  if (small_fwd(rows, inner, cols, pad_x || pad_w)) return 0;
  return (pad_x ? up(2 * padded(inner) * rows) : 0) + (pad_w ? up(2 * padded(inner) * cols) : 0);
}

extern "C" int aeris_linear_fwd(const AerisLinear* a, void* stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (a->rows <= 0 || a->inner <= 0 || a->cols <= 0 || !a->x || !a->w || !a->y || a->act < 0 || a->act > LIN_ACT_GELU_TANH) return -1;
  const bool pad_x = !tiled(a->x, a->ld_x, a->rows, a->inner), pad_w = !tiled(a->w, a->ld_w, a->cols, a->inner);
  if (a->work_bytes < aeris_linear_fwd_bytes(a->rows, a->inner, a->cols, pad_x, pad_w)) return -2;
  LinParams p{};
  p.M = a->rows; p.N = a->cols; p.K = a->inner; p.act = a->act; p.mode = LIN_OUT; p.k_splits = 1; p.bias_bf16 = a->bias_bf16;
  p.C = static_cast<__nv_bfloat16*>(a->y); p.ldc = pitch(a->ld_y, a->rows, a->cols); p.bias = a->bias;
  p.resid = static_cast<const __nv_bfloat16*>(a->resid); p.ldr = pitch(a->ld_resid, a->rows, a->cols);
  p.Z = static_cast<__nv_bfloat16*>(a->z); p.ldz = pitch(a->ld_z, a->rows, a->cols); p.status = a->status;
  int n = 1, r;
  if (small_fwd(a->rows, a->inner, a->cols, pad_x || pad_w)) {
    const int g = lanes_for(a->inner);
    r = launch_chained(lin_small_fwd_kernel, blocks_for(static_cast<long long>(a->rows) * a->cols * g), DZ_THREADS, 0, stream, p,
                       static_cast<const unsigned short*>(a->x), a->ld_x, static_cast<const unsigned short*>(a->w), a->ld_w, g);
    return r ? r : 1;
  }
  Operands operands{static_cast<uint8_t*>(a->work)};
  const Operand x = operands.add(a->x, a->ld_x, a->rows, a->inner), w = operands.add(a->w, a->ld_w, a->cols, a->inner);
  if ((r = operands.launch(n, stream))) return r;
  // x of few rows lies in shared memory, at most 48 KB of it
  if (a->rows <= ROWS_MAX && a->rows * padded(a->inner) * 2 <= 48 * 1024) r = launch_rows(p, x.p, x.ld, w.p, w.ld, stream);
  else r = launch_product<0, 0>(x.p, x.ld, w.p, w.ld, p, stream);
  return r ? r : n;
}

namespace {

// sx, sw: slices of dx's and dw's sums, 0 where it is not wanted.
long long bwd_bytes(int rows, int inner, int cols, bool own_dz, bool pad_x, bool pad_w, int sx, int sw, bool db, bool dw_f32) {
  const int slices = db ? db_slices(rows, cols) : 1;
  long long n = slices > 1 ? up(4ll * slices * cols) : 0;
  if (own_dz && (sx || sw)) n += up(2 * padded(cols) * rows);
  if (sx) n += (pad_w ? up(2 * padded(inner) * cols) : 0) + part_bytes(sx, rows, inner, false);
  if (sw) n += (pad_x ? up(2 * padded(inner) * rows) : 0) + part_bytes(sw, cols, inner, dw_f32);
  return n;
}

}  // namespace

extern "C" long long aeris_linear_bwd_bytes(int rows, int inner, int cols, int own_dz, int pad_x, int pad_w, int dx, int dw, int db,
                                            int dw_f32) {
  if (rows <= 0 || inner <= 0 || cols <= 0) return -1;
  if (small_bwd(rows, inner, cols)) return 0;
  return bwd_bytes(rows, inner, cols, own_dz, pad_x, pad_w, dx ? dx_slices(rows, inner, cols) : 0, dw ? dw_slices(rows, inner, cols) : 0, db,
                   dw_f32);
}

extern "C" int aeris_linear_bwd(const AerisLinearGrad* a, void* stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  const int rows = a->rows, inner = a->inner, cols = a->cols;
  if (rows <= 0 || inner <= 0 || cols <= 0 || !a->dy || a->act < 0 || a->act > LIN_ACT_GELU_TANH) return -1;
  if ((a->act != LIN_ACT_NONE) != (a->z != nullptr)) return -1;
  const bool products = a->dx || a->dw, own_dz = products && (a->z || !tiled(a->dy, a->ld_dy, rows, cols));
  int n = 0, r;
  if (small_bwd(rows, inner, cols)) {
    const long long results = (a->dx ? static_cast<long long>(rows) * inner : 0) + (a->dw ? static_cast<long long>(cols) * inner : 0) + cols;
    const int g = lanes_for(rows > cols ? rows : cols);
    r = launch_chained(lin_small_bwd_kernel, blocks_for(results * g), DZ_THREADS, 0, stream, *a, g);
    return r ? r : 1;
  }
  const int sx = a->dx ? dx_slices(rows, inner, cols) : 0, sw = a->dw ? dw_slices(rows, inner, cols) : 0;
  if (a->work_bytes < bwd_bytes(rows, inner, cols, own_dz, !tiled(a->x, a->ld_x, rows, inner), !tiled(a->w, a->ld_w, cols, inner), sx, sw,
                                a->db != nullptr, a->dw_f32))
    return -2;
  uint8_t* work = static_cast<uint8_t*>(a->work);
  long long at = 0;
  Operand dz{a->dy, pitch(a->ld_dy, rows, cols)};
  // [rows, inner] = dz [rows, cols] w [cols, inner], [cols, inner] = dz^T x
  LinBoth both{};
  LinParams &px = both.px, &pw = both.pw;
  px.M = rows; px.N = inner; px.K = cols; px.status = a->status;
  px.k_splits = sx;
  px.mode = px.k_splits > 1 ? LIN_PART : LIN_OUT;
  px.C = static_cast<__nv_bfloat16*>(a->dx); px.ldc = pitch(a->ld_dx, rows, inner);
  pw.M = cols; pw.N = inner; pw.K = rows; pw.status = a->status;
  pw.k_splits = sw;
  const bool direct = pw.k_splits == 1 && !a->dw_f32;
  pw.mode = direct ? LIN_OUT : LIN_PART;
  const int slices = db_slices(rows, cols), width = a->dx && a->dw ? both_width(px, pw) : 0;
  const bool db_beside = width && a->db && !own_dz && slices == 1;
  const dim3 dz_grid((cols + DZ_COLS - 1) / DZ_COLS, slices);
  if (own_dz || a->db) {
    DzParams& d = both.d;
    d = {a->dy, a->z, nullptr, nullptr, 0, a->ld_dy, a->ld_z, padded(cols), rows, cols};
    if (a->db && slices == 1) {
      d.sums = a->db;
      d.add = a->add_db;
    } else if (a->db) {
      d.sums = reinterpret_cast<float*>(work + at);
      at += up(4ll * slices * cols);
    }
    if (own_dz) {
      d.dz = work + at;
      dz = {d.dz, padded(cols)};
      at += up(2 * padded(cols) * rows);
    }
    both.d_vec = cols % 8 == 0 && whole_rows(d.dy, d.ld_dy) && (!d.z || whole_rows(d.z, d.ld_z));
    if (!db_beside) {
      if ((r = both.d_vec ? launch_dz<8>(d, a->act, dz_grid, stream) : launch_dz<1>(d, a->act, dz_grid, stream))) return r;
      ++n;
    }
    if (a->db && slices > 1) {
      r = launch_chained(lin_join_sums_kernel, (cols + 31) / 32, DZ_THREADS, 0, stream, static_cast<const float*>(d.sums), a->db, slices, cols,
                         a->add_db);
      if (r) return r;
      ++n;
    }
  }
  Operands operands{work, at};
  Operand w{}, x{};
  if (a->dx) w = operands.add(a->w, a->ld_w, cols, inner);
  if (a->dw) x = operands.add(a->x, a->ld_x, rows, inner);
  if ((r = operands.launch(n, stream))) return r;
  px.ld_part = pw.ld_part = (inner + 3) / 4 * 4;
  px.part = reinterpret_cast<float*>(work + operands.at);
  operands.at += part_bytes(sx, rows, inner, false);
  if (direct) {
    pw.C = static_cast<__nv_bfloat16*>(a->dw); pw.ldc = pitch(a->ld_dw, cols, inner);
  } else {
    pw.part = reinterpret_cast<float*>(work + operands.at);
  }
  auto join = [&](const LinParams& p, void* out, long long ld, int f32, int size) {
    const int vec = (reinterpret_cast<uintptr_t>(out) & 7) == 0 && ld % 4 == 0;
    ++n;
    return launch_chained(lin_join_kernel, blocks_for(static_cast<long long>(size) * ((inner + 3) / 4)), DZ_THREADS, 0, stream,
                          static_cast<const float*>(p.part), out, ld, f32, vec, p.k_splits, size, inner, p.ld_part);
  };
  if (width) {
    const int n_db = db_beside ? static_cast<int>(dz_grid.x) : 0;
    if ((r = width == 64 ? launch_both<64>(dz, w, x, both, n_db, stream) : launch_both<128>(dz, w, x, both, n_db, stream))) return r;
    ++n;
  } else {
    if (a->dx) {
      if ((r = launch_product<0, 1>(dz.p, dz.ld, w.p, w.ld, px, stream))) return r;
      ++n;
    }
    if (a->dw) {
      if ((r = launch_product<1, 1>(dz.p, dz.ld, x.p, x.ld, pw, stream))) return r - 1000;
      ++n;
    }
  }
  if (px.k_splits > 1 && (r = join(px, a->dx, px.ldc, 0, rows))) return r - 2000;
  if (a->dw && !direct && (r = join(pw, a->dw, a->ld_dw, a->dw_f32, cols))) return r - 2000;
  return n;
}
