// Linear layers of the plain block: products with bias, activation and residual in the epilogue, and their gradients.
//
//   z = x w^T + b, y = r + act(z)
//   dz = dy act'(z), db = sum dz, dx = dz w, dw = dz^T x                                    (sums over rows)
//
// Any number of rows and columns: operand tiles that reach past a matrix are filled with zeros by the tensor maps, results
// past it are clipped by them or, where rows do not start on 16-byte boundaries, masked element by element. fp32 accumulation;
// bias, activation and residual are applied to the accumulators, which are rounded once.
#include "common.cuh"
#include "api.h"
#include "host.h"
#include "gemm_epilogue.cuh"

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

// Gaussian distribution function. erff is CUDA's; near -infinity the sum cancels to an absolute error of 6e-8.
__device__ __forceinline__ float gauss_cdf(float z) { return fmaf(0.5f, erff(z * 0.70710678118654752f), 0.5f); }
__device__ __forceinline__ float sigmoid(float z) { return 1.f / (1.f + __expf(-z)); }

// gelu_tanh by 0.5 (1 + tanh u) = 1 / (1 + exp(-2 u)), which keeps the relative precision of small results.
__device__ __forceinline__ float act_of(float z, int act) {
  switch (act) {
    case LIN_ACT_RELU: return z < 0.f ? 0.f : z;      // a NaN stays
    case LIN_ACT_SILU: return z * sigmoid(z);
    case LIN_ACT_GELU: return z * gauss_cdf(z);
    case LIN_ACT_GELU_TANH: return z * sigmoid(z * fmaf(z * z, 0.07135481282f, 1.59576912161f));
    default: return z;
  }
}
__device__ __forceinline__ float act_grad(float z, int act) {
  switch (act) {
    case LIN_ACT_RELU: return z > 0.f ? 1.f : 0.f;
    case LIN_ACT_SILU: { const float s = sigmoid(z); return s * fmaf(z, 1.f - s, 1.f); }
    case LIN_ACT_GELU: return fmaf(z * 0.39894228040143268f, __expf(-0.5f * z * z), gauss_cdf(z));
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
// unit as 32 x 32 tiles (64-byte swizzle); what lies past the matrix is clipped.
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

// The first `n` of 32 bf16 columns of one row, element by element: rows that start anywhere.
__device__ __forceinline__ void store_row32(__nv_bfloat16* dst, const uint32_t (&o)[16], int n) {
#pragma unroll
  for (int i = 0; i < 32; ++i)
    if (i < n) {
      const uint32_t h = i & 1 ? o[i / 2] >> 16 : o[i / 2] & 0xffffu;
      reinterpret_cast<unsigned short*>(dst)[i] = static_cast<unsigned short>(h);
    }
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
      else if (row_ok) store_row32(p.Z + static_cast<long long>(row) * p.ldz + col0 + c, o, n);
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
    else if (row_ok) store_row32(p.C + static_cast<long long>(row) * p.ldc + col0 + c, o, n);
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

template <int BN, int A_MN, int B_MN>
__global__ void __launch_bounds__(LIN_THREADS, 1)
lin_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
           const __grid_constant__ CUtensorMap tm_y, const __grid_constant__ CUtensorMap tm_z, const LinParams p) {
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
      for (int tile = blockIdx.x; tile < total_tiles && ok; tile += gridDim.x) {
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
      for (int tile = blockIdx.x; tile < total_tiles && ok; tile += gridDim.x) {
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
  } else {
    const int q = warp & 3;  // TMEM lane quarter this warp may access
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    const bool keep = !failed(p.status);       // see note_failure
    LinOut out{smem + S::OUT + q * 8192, lane};
    for (int tile = blockIdx.x; tile < total_tiles && ok; tile += gridDim.x) {
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

bool whole_rows(const void* base, long long ld) { return (reinterpret_cast<uintptr_t>(base) & 15) == 0 && ld % 8 == 0; }

template <int BN, int A_MN, int B_MN>
int launch_lin(const void* A, long long lda, const void* B, long long ldb, LinParams p, cudaStream_t stream) {
  using S = LinSmem<BN>;
  auto kern = lin_kernel<BN, A_MN, B_MN>;
  static std::atomic<uint64_t> done{0};
  if (!allow_smem_once(kern, S::TOTAL, done)) return -20;
  CUtensorMap ta, tb, ty, tz;
  int r;
  if (!whole_rows(A, lda) || !whole_rows(B, ldb)) return -11;
  if ((r = A_MN ? make_tmap_2d_bf16(&ta, A, p.M, p.K, lda, 64, LIN_BK) : make_tmap_2d_bf16(&ta, A, p.K, p.M, lda, LIN_BK, LIN_BM)))
    return r;
  if ((r = B_MN ? make_tmap_2d_bf16(&tb, B, p.N, p.K, ldb, 64, LIN_BK) : make_tmap_2d_bf16(&tb, B, p.K, p.N, ldb, LIN_BK, BN)))
    return r - 100;
  ty = tz = ta;         // not stored through where rows go element by element
  p.c_map = p.mode == LIN_OUT && whole_rows(p.C, p.ldc);
  p.z_map = p.mode == LIN_OUT && p.Z && whole_rows(p.Z, p.ldz);
  p.r_vec = p.resid && whole_rows(p.resid, p.ldr);
  if (p.c_map && (r = make_tmap_2d_sw64_bf16(&ty, p.C, p.N, p.M, p.ldc, 32, 32))) return r - 200;
  if (p.z_map && (r = make_tmap_2d_sw64_bf16(&tz, p.Z, p.N, p.M, p.ldz, 32, 32))) return r - 300;
  const long long tiles = static_cast<long long>((p.M + LIN_BM - 1) / LIN_BM) * ((p.N + BN - 1) / BN) * p.k_splits;
  if (tiles > 0x3fffffff) return -2;
  const int grid = tiles < num_sms() ? static_cast<int>(tiles) : num_sms();
  return launch_chained(kern, grid, LIN_THREADS, S::TOTAL, stream, ta, tb, ty, tz, p);
}

long long lin_tiles(int M, int N, int bn) { return static_cast<long long>((M + LIN_BM - 1) / LIN_BM) * ((N + bn - 1) / bn); }

// Width of the tiles: the widest of which there is one for every multiprocessor, else narrow ones.
template <int A_MN, int B_MN>
int launch_product(const void* A, long long lda, const void* B, long long ldb, const LinParams& p, cudaStream_t stream) {
  if (lin_tiles(p.M, p.N, 256) * p.k_splits >= num_sms()) return launch_lin<256, A_MN, B_MN>(A, lda, B, ldb, p, stream);
  if (lin_tiles(p.M, p.N, 128) * p.k_splits >= num_sms()) return launch_lin<128, A_MN, B_MN>(A, lda, B, ldb, p, stream);
  if constexpr (!B_MN) {
    if (lin_tiles(p.M, p.N, 64) * p.k_splits < num_sms()) return launch_lin<32, A_MN, B_MN>(A, lda, B, ldb, p, stream);
  }
  return launch_lin<64, A_MN, B_MN>(A, lda, B, ldb, p, stream);
}

// ------------------------------------------------------------------------------------------------ gradients' own passes
constexpr int DZ_THREADS = 256, DZ_COLS = 64;

__device__ __forceinline__ float bf(unsigned short u) { return __uint_as_float(static_cast<uint32_t>(u) << 16); }

// dz = dy act'(z) and the column sums of one slice of the rows. A thread takes V columns (one 16-byte vector, or one column
// where rows start anywhere) of every R-th row of its slice; a block 64 columns.
template <int V>
__global__ void __launch_bounds__(DZ_THREADS) lin_dz_kernel(const AerisLinearDz a) {
  constexpr int CT = DZ_COLS / V, R = DZ_THREADS / CT;
  __shared__ float part[R][DZ_COLS];
  chain_point();
  const int c0 = threadIdx.x % CT * V, col = blockIdx.x * DZ_COLS + c0, r0 = threadIdx.x / CT;
  float s[V] = {};
  if (col < a.cols) {
    for (long long row = static_cast<long long>(blockIdx.y) * R + r0; row < a.rows; row += static_cast<long long>(gridDim.y) * R) {
      const unsigned short* dy = static_cast<const unsigned short*>(a.dy) + row * a.ld_dy + col;
      const unsigned short* z = a.z ? static_cast<const unsigned short*>(a.z) + row * a.ld_z + col : nullptr;
      unsigned short d[V], zz[V];
      if constexpr (V == 8) {
        *reinterpret_cast<uint4*>(d) = *reinterpret_cast<const uint4*>(dy);
        if (z) *reinterpret_cast<uint4*>(zz) = *reinterpret_cast<const uint4*>(z);
      } else {
        d[0] = *dy;
        if (z) zz[0] = *z;
      }
      float g[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        // a product by itself, so that the sums are the same bits whether dz is written or not
        g[i] = z ? __fmul_rn(bf(d[i]), act_grad(bf(zz[i]), a.act)) : bf(d[i]);
        s[i] += g[i];
      }
      if (a.dz) {
        __nv_bfloat16* dz = static_cast<__nv_bfloat16*>(a.dz) + row * a.ld_dz + col;
        if constexpr (V == 8)
          *reinterpret_cast<uint4*>(dz) = make_uint4(pack_bf16x2(g[0], g[1]), pack_bf16x2(g[2], g[3]), pack_bf16x2(g[4], g[5]),
                                                     pack_bf16x2(g[6], g[7]));
        else
          *dz = __float2bfloat16_rn(g[0]);
      }
    }
  }
  if (!a.db) return;
#pragma unroll
  for (int i = 0; i < V; ++i) part[r0][c0 + i] = s[i];
  __syncthreads();
  if (threadIdx.x < DZ_COLS && blockIdx.x * DZ_COLS + threadIdx.x < a.cols) {
    float t = 0.f;
    for (int r = 0; r < R; ++r) t += part[r][threadIdx.x];
    a.work[static_cast<long long>(blockIdx.y) * a.cols + blockIdx.x * DZ_COLS + threadIdx.x] = t;
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

// dw from the sums of slices of the rows, in their order. `part`: [slices, rows, ld] fp32, ld a multiple of 4.
__global__ void __launch_bounds__(DZ_THREADS) lin_join_dw_kernel(const float* part, void* dw, long long ld_dw, int f32, int vec,
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

// Slices of the reduction over the rows of dw: enough tiles for every multiprocessor, rounds x (k-blocks of a slice + 10 for its
// start and its sums); at most 8192 rows a slice, for the tensor core truncates at every addition and the error of a sum grows
// with its length (9e-10 of it per row).
int dw_slices(int rows, int inner, int cols) {
  const int kb = (rows + LIN_BK - 1) / LIN_BK;
  const long long tiles = lin_tiles(cols, inner, 256);
  int best = (kb + 127) / 128;
  auto cost = [&](int s) { return ((tiles * s + num_sms() - 1) / num_sms()) * ((kb + s - 1) / s + 10); };
  for (int s = best + 1; s <= 64 && kb / s >= 4; ++s)
    if (cost(s) < cost(best)) best = s;
  return best;
}

}  // namespace

}  // namespace aeris

using namespace aeris;

extern "C" int aeris_linear_fwd(const AerisLinear* a, void* stream_) {
  if (a->rows <= 0 || a->inner <= 0 || a->cols <= 0 || !a->y || a->act < 0 || a->act > LIN_ACT_GELU_TANH) return -1;
  LinParams p{};
  p.M = a->rows; p.N = a->cols; p.K = a->inner; p.act = a->act; p.mode = LIN_OUT; p.k_splits = 1; p.bias_bf16 = a->bias_bf16;
  p.C = static_cast<__nv_bfloat16*>(a->y); p.ldc = a->ld_y; p.bias = a->bias;
  p.resid = static_cast<const __nv_bfloat16*>(a->resid); p.ldr = a->ld_resid;
  p.Z = static_cast<__nv_bfloat16*>(a->z); p.ldz = a->ld_z; p.status = a->status;
  const int r = launch_product<0, 0>(a->x, a->ld_x, a->w, a->ld_w, p, static_cast<cudaStream_t>(stream_));
  return r ? r : 1;
}

extern "C" int aeris_linear_dz(const AerisLinearDz* a, void* stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (a->rows <= 0 || a->cols <= 0 || !a->dy || (!a->dz && !a->db) || a->slices <= 0 || a->slices > 65535) return -1;
  if (a->db && !a->work) return -2;
  const bool vec = a->cols % 8 == 0 && whole_rows(a->dy, a->ld_dy) && (!a->z || whole_rows(a->z, a->ld_z)) &&
                   (!a->dz || whole_rows(a->dz, a->ld_dz));
  const dim3 grid((a->cols + DZ_COLS - 1) / DZ_COLS, a->slices);
  int r = vec ? launch_chained(lin_dz_kernel<8>, grid, DZ_THREADS, 0, stream, *a)
              : launch_chained(lin_dz_kernel<1>, grid, DZ_THREADS, 0, stream, *a);
  if (r) return r;
  if (!a->db) return 1;
  r = launch_chained(lin_join_sums_kernel, (a->cols + 31) / 32, DZ_THREADS, 0, stream, static_cast<const float*>(a->work), a->db,
                     a->slices, a->cols, a->add);
  return r ? r : 2;
}

extern "C" long long aeris_linear_work_bytes(int rows, int inner, int cols, int dw_f32) {
  if (rows <= 0 || inner <= 0 || cols <= 0) return -1;
  const int s = dw_slices(rows, inner, cols);
  return s > 1 || dw_f32 ? 4ll * s * cols * ((inner + 3) / 4 * 4) : 0;
}

extern "C" int aeris_linear_grad(const AerisLinearGrad* a, void* stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (a->rows <= 0 || a->inner <= 0 || a->cols <= 0 || (!a->dx && !a->dw)) return -1;
  int n = 0, r;
  if (a->dx) {        // [rows, inner] = dz [rows, cols] w [cols, inner]
    LinParams p{};
    p.M = a->rows; p.N = a->inner; p.K = a->cols; p.mode = LIN_OUT; p.k_splits = 1;
    p.C = static_cast<__nv_bfloat16*>(a->dx); p.ldc = a->ld_dx; p.status = a->status;
    if ((r = launch_product<0, 1>(a->dz, a->ld_dz, a->w, a->ld_w, p, stream))) return r;
    ++n;
  }
  if (a->dw) {        // [cols, inner] = dz^T x
    LinParams p{};
    p.M = a->cols; p.N = a->inner; p.K = a->rows; p.status = a->status;
    p.k_splits = dw_slices(a->rows, a->inner, a->cols);
    const bool direct = p.k_splits == 1 && !a->dw_f32;
    p.mode = direct ? LIN_OUT : LIN_PART;
    if (direct) {
      p.C = static_cast<__nv_bfloat16*>(a->dw); p.ldc = a->ld_dw;
    } else {
      if (!a->work || a->work_bytes < aeris_linear_work_bytes(a->rows, a->inner, a->cols, a->dw_f32)) return -3;
      p.part = a->work; p.ld_part = (a->inner + 3) / 4 * 4;
    }
    if ((r = launch_product<1, 1>(a->dz, a->ld_dz, a->x, a->ld_x, p, stream))) return r - 1000;
    ++n;
    if (!direct) {
      const long long vecs = static_cast<long long>(a->cols) * ((a->inner + 3) / 4);
      const long long blocks = (vecs + DZ_THREADS - 1) / DZ_THREADS;
      const int vec = (reinterpret_cast<uintptr_t>(a->dw) & 7) == 0 && a->ld_dw % 4 == 0;
      r = launch_chained(lin_join_dw_kernel, static_cast<unsigned>(blocks < 16 * num_sms() ? blocks : 16 * num_sms()), DZ_THREADS, 0,
                         stream, static_cast<const float*>(a->work), a->dw, a->ld_dw, a->dw_f32, vec, p.k_splits, a->cols, a->inner,
                         p.ld_part);
      if (r) return r - 2000;
      ++n;
    }
  }
  return n;
}
