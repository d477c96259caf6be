// Learned bias by relative position in window attention: what stands around the attention kernels (attention.cu), and the
// gradient of the table.
//
//   s_ij = scale q_i k_j + table[bucket(pos_i - pos_j), head], p = softmax_j(s), o = p v
//   ds = p (dp - delta), dp = dO v^T, delta = rowsum(p dp);  dtable[b, head] = sum of ds over windows and the pairs of bucket b
//
// The bias of a pair is a function of the difference of two tokens' places: with at(t) = y (2 wide - 1) + x it is entry
// at(i) - at(j) + at(last) of a table by relative position, which is all that the attention kernels read: one table of
// (2 high - 1)(2 wide - 1) floats for a head, whatever the buckets, in log2 units, instead of an N x N matrix.
#include "common.cuh"
#include "api.h"
#include "host.h"

#include <atomic>

namespace aeris {

namespace {

constexpr float HIDDEN = -1e30f;
constexpr int PB_TILE = 128;

struct Place {
  int n, off;         // tokens of a window, relative positions
  int at_words;       // `at`, up to the next multiple of 128 behind the window's end
};
Place place_of(int high, int wide) {
  Place p;
  p.n = high * wide;
  p.off = (2 * high - 1) * (2 * wide - 1);
  p.at_words = (p.n + 127) / 128 * 128;
  return p;
}

// The table by relative position [heads, off] in log2 units, and the places of the tokens.
__global__ void __launch_bounds__(256) bias_expand_kernel(const AerisBiasedAttn a, float* out, int* at, int n, int off, int at_words) {
  chain_point();
  const int i = blockIdx.x * 256 + threadIdx.x, head = blockIdx.y;
  if (i < off) {
    long long b = i;
    if (a.buckets)
      b = a.buckets64 ? static_cast<const long long*>(a.buckets)[i] : static_cast<const int*>(a.buckets)[i];
    float v = -INFINITY;
    if (b >= 0 && b < a.table_rows) {
      const long long k = b * a.heads + head;
      v = a.table_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(a.table)[k]) : static_cast<const float*>(a.table)[k];
      v = v <= HIDDEN ? -INFINITY : v * 1.4426950408889634f;
    } else if (a.status) {
      atomicCAS(a.status, 0, ERR_BOUNDS);
    }
    out[static_cast<long long>(head) * off + i] = v;
  }
  if (head == 0 && i < at_words) {
    const int t = i < n ? i : n - 1, y = t / a.wide;
    at[i] = y * (2 * a.wide - 1) + t - y * a.wide;
  }
}

// ------------------------------------------------------------------------------------------ sums of dS over windows
// One CTA = a 128 x TK tile of (query, key) of one head. It goes over its windows: S = Q K^T and dP = dO V^T into TMEM, two
// buffers in turn, and adds p (dp - delta) to sums that stay in registers; the bias of its pairs stays there too. No atomics: slices of
// the windows have sums of their own, which bias_sums_kernel adds in their order.
template <int DCH> struct BgCfg {
  static constexpr int TK = DCH == 1 ? 128 : 64, CPT = TK / 4;
  static constexpr int QB = DCH * 16384, KB = DCH * TK * 128, STAGE = 2 * QB + 2 * KB, NST = DCH == 1 ? 3 : 2;
  static constexpr int MATH = 16, THREADS = 64 + 32 * MATH;
  static constexpr int TMEM = 4 * TK, SMEM = NST * STAGE + 256 + 1024;
  static_assert(SMEM <= 227 * 1024, "shared memory");
};

struct BgParams {
  const float *lse, *delta, *table;
  const int* at;
  float* part;                // [splits, heads at hand, n, ld]
  long long ld;
  int n, heads, n_win, off, zero, head0, n_heads, splits;
  float scale_log2;
  int* status;
};

__device__ __forceinline__ float bg_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <int DCH>
__global__ void __launch_bounds__(BgCfg<DCH>::THREADS, 1)
bias_grad_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_do,
                 const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const BgParams p) {
  using C = BgCfg<DCH>;
  constexpr int TK = C::TK, CPT = C::CPT, NST = C::NST;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + NST * C::STAGE);     // [NST]
  uint64_t* empty = full + NST;
  uint64_t* s_full = empty + NST;       // [2]
  uint64_t* s_empty = s_full + 2;       // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(s_empty + 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  {
    __shared__ int s_abort;
    if (threadIdx.x == 0) s_abort = failed(p.status) ? 1 : 0;
    __syncthreads();
    if (s_abort) { chain_point(); return; }
  }
  const int ti = blockIdx.x, tj = blockIdx.y, split = blockIdx.z / p.n_heads, hl = blockIdx.z - split * p.n_heads;
  const int head = p.head0 + hl, per = (p.n_win + p.splits - 1) / p.splits;
  const int w0 = split * per, w1 = min(p.n_win, w0 + per);
  if (threadIdx.x == 0) {
    prefetch_tmap(&tm_q); prefetch_tmap(&tm_do); prefetch_tmap(&tm_k); prefetch_tmap(&tm_v);
    for (int i = 0; i < NST; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(&s_full[i], 1); mbar_init(&s_empty[i], C::MATH); }
    fence_barrier_init();
  }
  if (warp == 1) { tmem_alloc(tmem_slot, C::TMEM); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  chain_point();

  if (warp == 0) {
    if (elect_one_sync()) {
      int st = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int w = w0; w < w1; ++w) {
        if (!mbar_wait(&empty[st], ph ^ 1, p.status, ERR_TIMEOUT_ATTN)) { ok = false; break; }
        uint8_t* s = smem + st * C::STAGE;
        mbar_expect_tx(&full[st], C::STAGE);
#pragma unroll
        for (int c = 0; c < DCH; ++c) {
          tma_load_4d(s + c * 16384, &tm_q, &full[st], c * 64, head, ti * PB_TILE, w);
          tma_load_4d(s + 2 * C::QB + c * (TK * 128), &tm_k, &full[st], c * 64, head, tj * TK, w);
          tma_load_4d(s + C::QB + c * 16384, &tm_do, &full[st], c * 64, head, ti * PB_TILE, w);
          tma_load_4d(s + 2 * C::QB + C::KB + c * (TK * 128), &tm_v, &full[st], c * 64, head, tj * TK, w);
        }
        if (++st == NST) { st = 0; ph ^= 1; }
      }
      for (int i = 0; i < NST && ok; ++i) {      // every stage has been released: no copy is under way at exit
        ok = mbar_wait(&empty[st], ph ^ 1, p.status, ERR_TIMEOUT_ATTN);
        if (++st == NST) { st = 0; ph ^= 1; }
      }
    }
  } else if (warp == 1) {
    if (elect_one_sync()) {
      constexpr uint32_t idesc = make_idesc_bf16(PB_TILE, TK, 0, 0);
      int st = 0, buf = 0;
      uint32_t ph = 0, bph = 0;
      for (int w = w0; w < w1; ++w) {
        if (!mbar_wait(&s_empty[buf], bph ^ 1, p.status, ERR_TIMEOUT_ATTN)) break;
        if (!mbar_wait(&full[st], ph, p.status, ERR_TIMEOUT_ATTN)) break;
        tc_fence_after();
        const uint32_t s = smem_u32(smem + st * C::STAGE), t = tmem_base + buf * 2 * TK;
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int kk = 0; kk < 4 * DCH; ++kk)
            umma_ss(t + m * TK, make_smem_desc(s + m * C::QB + (kk >> 2) * 16384 + (kk & 3) * 32, 0, 1024),
                    make_smem_desc(s + 2 * C::QB + m * C::KB + (kk >> 2) * (TK * 128) + (kk & 3) * 32, 0, 1024), idesc, kk > 0);
        tc_commit(&empty[st]);
        tc_commit(&s_full[buf]);
        if (++st == NST) { st = 0; ph ^= 1; }
        if (++buf == 2) { buf = 0; bph ^= 1; }
      }
    }
  } else {
    const int q = warp & 3, g = (warp - 2) >> 2;
    const int row = ti * PB_TILE + q * 32 + lane, col = tj * TK + g * CPT;      // of this thread's sums
    const bool in = row < p.n;
    const uint32_t t0 = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + g * CPT;
    float bias[CPT], sum[CPT];
    {
      const float* b = p.table + static_cast<long long>(head) * p.off + p.zero + p.at[in ? row : p.n - 1];
#pragma unroll
      for (int i = 0; i < CPT; ++i) {
        bias[i] = col + i < p.n ? b[-p.at[col + i]] : -INFINITY;
        sum[i] = 0.f;
      }
    }
    const long long base = static_cast<long long>(head) * p.n + (in ? row : 0), step = static_cast<long long>(p.heads) * p.n;
    int buf = 0;
    uint32_t bph = 0;
    bool ok = true;
    float lse = w0 < w1 ? p.lse[base + w0 * step] : 0.f, delta = w0 < w1 ? p.delta[base + w0 * step] : 0.f;
    for (int w = w0; w < w1; ++w) {
      const float l = lse, d = delta;
      if (w + 1 < w1) {
        lse = p.lse[base + (w + 1) * step];
        delta = p.delta[base + (w + 1) * step];
      }
      if (!mbar_wait_warp(&s_full[buf], bph, p.status, ERR_TIMEOUT_ATTN)) { ok = false; break; }
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < CPT; c += 16) {
        uint32_t s[16], dp[16];
        tmem_ld16(t0 + buf * 2 * TK + c, s);
        tmem_ld16(t0 + buf * 2 * TK + TK + c, dp);
        tmem_wait_ld();
        if (c + 16 == CPT) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s_empty[buf]);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float e = bg_exp2(fmaf(__uint_as_float(s[i]), p.scale_log2, bias[c + i]) - l);
          sum[c + i] = fmaf(e, __uint_as_float(dp[i]) - d, sum[c + i]);
        }
      }
      if (++buf == 2) { buf = 0; bph ^= 1; }
    }
    if (ok && in && !failed(p.status)) {
      float* dst = p.part + ((static_cast<long long>(split) * p.n_heads + hl) * p.n + row) * p.ld + col;       // ld a multiple of 4
#pragma unroll
      for (int i = 0; i < CPT; i += 4)
        if (col + i < p.n) *reinterpret_cast<float4*>(dst + i) = make_float4(sum[i], sum[i + 1], sum[i + 2], sum[i + 3]);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem_base, C::TMEM);
}

// Sums of the pairs of one relative position: a block has 32 positions of one difference in y (a lane each), its warps
// share the queries. Lanes read neighbouring keys of one query: 128 bytes a load.
__global__ void __launch_bounds__(256) bias_sums_kernel(const float* part, long long ld, int splits, int n_heads, int head0, int high,
                                                        int wide, float* out, int heads, int add) {
  __shared__ float part_sum[8][32];
  chain_point();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int dy = static_cast<int>(blockIdx.x) - (high - 1), k = blockIdx.y * 32 + lane, dx = k - (wide - 1), hl = blockIdx.z;
  const int n = high * wide, y0 = max(0, dy), y1 = min(high, high + dy), rows = (y1 - y0) * wide;
  float s = 0.f;
  for (int sp = 0; sp < splits; ++sp) {
    const float* src = part + (static_cast<long long>(sp) * n_heads + hl) * n * ld;
#pragma unroll 4
    for (int r = warp; r < rows; r += 8) {
      const int y = y0 + r / wide, xi = r % wide, xj = xi - dx;
      if (xj >= 0 && xj < wide) s += src[static_cast<long long>(y * wide + xi) * ld + (y - dy) * wide + xj];
    }
  }
  part_sum[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && k < 2 * wide - 1) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += part_sum[i][lane];
    float* dst = out + static_cast<long long>(blockIdx.x * (2 * wide - 1) + k) * heads + head0 + hl;
    *dst = add ? *dst + s : s;
  }
}

// Sums of the relative positions of one bucket: a block per bucket and 32 heads; its warps share the positions.
__global__ void __launch_bounds__(256) bias_buckets_kernel(const AerisBiasedAttn a, const float* by_position, int off) {
  __shared__ float part_sum[8][32];
  chain_point();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, b = blockIdx.x, head = blockIdx.y * 32 + lane;
  float s = 0.f;
#pragma unroll 4
  for (int i = warp; i < off; i += 8) {
    const long long k = a.buckets64 ? static_cast<const long long*>(a.buckets)[i] : static_cast<const int*>(a.buckets)[i];
    if (k == b && head < a.heads) s += by_position[static_cast<long long>(i) * a.heads + head];
  }
  part_sum[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && head < a.heads) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += part_sum[i][lane];
    float* dst = a.dtable + static_cast<long long>(b) * a.heads + head;
    *dst = a.add ? *dst + s : s;
  }
}

__global__ void __launch_bounds__(256) bias_zero_kernel(float* p, long long n) {
  chain_point();
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n; i += 256ll * gridDim.x) p[i] = 0.f;
}

// Lets a kernel have `bytes` of shared memory, once a device.
template <typename F> bool allow_smem(F kernel, int bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  const uint64_t bit = 1ull << (dev & 63);
  if (done.load(std::memory_order_relaxed) & bit) return true;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
  done.fetch_or(bit, std::memory_order_relaxed);
  return true;
}

constexpr long long PART_BYTES = 256ll << 20;

// How the sums of dS are taken: slices of the windows, heads at a time (their matrices take at most 256 MB, or are one head's).
struct SumsPlan {
  int splits, heads;
  long long ld, bytes;
};
SumsPlan plan_sums(int n_win, int n, int heads, int head_dim) {
  SumsPlan s;
  s.ld = (n + 3) / 4 * 4;
  const int tk = head_dim <= 64 ? BgCfg<1>::TK : BgCfg<2>::TK;
  const long long tiles = static_cast<long long>((n + PB_TILE - 1) / PB_TILE) * ((n + tk - 1) / tk) * heads;
  // a slice costs as much as four windows to start and to add up
  auto cost = [&](long long k) { return (tiles * k + num_sms() - 1) / num_sms() * ((n_win + k - 1) / k + 4); };
  s.splits = 1;
  for (int k = 2; k <= n_win && k <= 64; ++k)
    if (cost(k) < cost(s.splits)) s.splits = k;
  const long long one = 4ll * s.splits * n * s.ld;
  s.heads = static_cast<int>(PART_BYTES / one);
  if (s.heads < 1) s.heads = 1;
  if (s.heads > heads) s.heads = heads;
  while (s.heads > 1 && static_cast<long long>(s.heads) * s.splits > 65535) --s.heads;
  s.bytes = one * s.heads;
  return s;
}

long long up(long long bytes) { return (bytes + 255) / 256 * 256; }

struct Work {
  long long table, at, delta, rest, by_position, part, total;
};
Work work_of(int n_win, int high, int wide, int heads, int head_dim, bool backward, bool with_table) {
  const Place p = place_of(high, wide);
  Work w{};
  const long long stats = 4ll * n_win * heads * p.n;
  w.at = up(4ll * heads * p.off);
  w.delta = w.at + up(4ll * p.at_words);
  w.rest = w.delta + (backward ? up(stats) : 0);
  w.by_position = w.rest + (backward ? up(4 * stats) : 0);
  w.part = w.by_position + (backward && with_table ? up(4ll * heads * p.off) : 0);
  w.total = w.part + (backward && with_table ? up(plan_sums(n_win, p.n, heads, head_dim).bytes) : 0);
  return w;
}

bool fits(const AerisBiasedAttn* a) {
  return a->n_win > 0 && a->high > 0 && a->wide > 0 && a->heads > 0 && a->head_dim > 0 && a->n_win <= 65535 && a->heads <= 65535 &&
         a->high <= 32768 && a->wide <= 32768 && static_cast<long long>(a->high) * a->wide <= 32768 && a->table && a->table_rows > 0 &&
         a->work && (reinterpret_cast<uintptr_t>(a->work) & 255) == 0 && a->ld_qkv <= 0x7fffffff && a->ld_o <= 0x7fffffff &&
         a->ld_dqkv <= 0x7fffffff;
}

int expand(const AerisBiasedAttn* a, const Place& p, float* table, int* at, cudaStream_t stream) {
  const int most = p.off > p.at_words ? p.off : p.at_words;
  return launch_chained(bias_expand_kernel, dim3((most + 255) / 256, a->heads), 256, 0, stream, *a, table, at, p.n, p.off, p.at_words);
}

template <int DCH>
int launch_bias_grad(const CUtensorMap (&m)[4], const BgParams& p, dim3 grid, cudaStream_t stream) {
  static std::atomic<uint64_t> done{0};
  if (!allow_smem(bias_grad_kernel<DCH>, BgCfg<DCH>::SMEM, done)) return -20;
  return launch_chained(bias_grad_kernel<DCH>, grid, BgCfg<DCH>::THREADS, BgCfg<DCH>::SMEM, stream, m[0], m[1], m[2], m[3], p);
}

}  // namespace

}  // namespace aeris

using namespace aeris;

extern "C" long long aeris_biased_attn_work_bytes(int n_win, int high, int wide, int heads, int head_dim, int backward, int with_table) {
  if (n_win <= 0 || high <= 0 || wide <= 0 || heads <= 0 || head_dim <= 0 || static_cast<long long>(high) * wide > 32768) return -1;
  return work_of(n_win, high, wide, heads, head_dim, backward, with_table).total;
}

extern "C" int aeris_biased_attn_fwd(const AerisBiasedAttn* a, void* stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (!fits(a)) return -1;
  const Work w = work_of(a->n_win, a->high, a->wide, a->heads, a->head_dim, false, false);
  if (a->work_bytes < w.total) return -2;
  const Place p = place_of(a->high, a->wide);
  uint8_t* work = static_cast<uint8_t*>(a->work);
  float* table = reinterpret_cast<float*>(work + w.table);
  int* at = reinterpret_cast<int*>(work + w.at);
  int r = expand(a, p, table, at, stream);
  if (r) return r;
  r = attn_fwd_biased(a->qkv, static_cast<int>(a->ld_qkv), a->o, static_cast<int>(a->ld_o), a->lse, a->n_win, p.n, a->heads, a->head_dim,
                      a->scale, table, at, p.off, p.off / 2, a->status, stream);
  return r ? r - 100 : 2;
}

extern "C" int aeris_biased_attn_bwd(const AerisBiasedAttn* a, void* stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (!fits(a) || !a->d_o || !a->dqkv || !a->lse) return -1;
  const bool sums = a->dtable != nullptr;
  const Work w = work_of(a->n_win, a->high, a->wide, a->heads, a->head_dim, true, sums);
  if (a->work_bytes < w.total) return -2;
  const Place p = place_of(a->high, a->wide);
  uint8_t* work = static_cast<uint8_t*>(a->work);
  float* table = reinterpret_cast<float*>(work + w.table);
  int* at = reinterpret_cast<int*>(work + w.at);
  float* delta = reinterpret_cast<float*>(work + w.delta);
  int r = expand(a, p, table, at, stream);
  if (r) return r;
  r = attn_bwd_biased(a->qkv, static_cast<int>(a->ld_qkv), a->o, a->d_o, static_cast<int>(a->ld_o), a->lse, delta,
                      reinterpret_cast<float*>(work + w.rest), a->dqkv, static_cast<int>(a->ld_dqkv), a->n_win, p.n, a->heads,
                      a->head_dim, a->scale, table, at, p.off, p.off / 2, a->status, stream);
  if (r) return r - 100;
  int count = 4;
  if (!sums) return count;
  if (p.n == 1) {       // one token sees itself whatever the bias
    if (a->add) return count;
    const long long cells = static_cast<long long>(a->table_rows) * a->heads, blocks = (cells + 255) / 256;
    r = launch_chained(bias_zero_kernel, static_cast<unsigned>(blocks < 1024 ? blocks : 1024), 256, 0, stream, a->dtable, cells);
    return r ? r : count + 1;
  }
  const int dch = a->head_dim <= 64 ? 1 : 2, tk = dch == 1 ? BgCfg<1>::TK : BgCfg<2>::TK, hd = a->heads * a->head_dim;
  const __nv_bfloat16* b = static_cast<const __nv_bfloat16*>(a->qkv);
  CUtensorMap m[4];
  const struct { const void* base; long long ld; uint32_t rows; } ops[4] = {
      {b, a->ld_qkv, PB_TILE}, {a->d_o, a->ld_o, PB_TILE}, {b + hd, a->ld_qkv, static_cast<uint32_t>(tk)},
      {b + 2 * hd, a->ld_qkv, static_cast<uint32_t>(tk)}};
  for (int i = 0; i < 4; ++i)
    if ((r = make_tmap_heads_bf16(&m[i], ops[i].base, a->head_dim, a->heads, p.n, a->n_win, ops[i].ld, ops[i].rows))) return r - 200;
  const SumsPlan s = plan_sums(a->n_win, p.n, a->heads, a->head_dim);
  BgParams g{};
  g.lse = a->lse; g.delta = delta; g.table = table; g.at = at; g.part = reinterpret_cast<float*>(work + w.part); g.ld = s.ld;
  g.n = p.n; g.heads = a->heads; g.n_win = a->n_win; g.off = p.off; g.zero = p.off / 2; g.splits = s.splits;
  g.scale_log2 = a->scale * 1.4426950408889634f; g.status = a->status;
  float* by_position = a->buckets ? reinterpret_cast<float*>(work + w.by_position) : a->dtable;
  for (int h0 = 0; h0 < a->heads; h0 += s.heads) {
    g.head0 = h0;
    g.n_heads = a->heads - h0 < s.heads ? a->heads - h0 : s.heads;
    const dim3 grid((p.n + PB_TILE - 1) / PB_TILE, (p.n + tk - 1) / tk, s.splits * g.n_heads);
    if ((r = dch == 1 ? launch_bias_grad<1>(m, g, grid, stream) : launch_bias_grad<2>(m, g, grid, stream))) return r - 300;
    r = launch_chained(bias_sums_kernel, dim3(2 * a->high - 1, (2 * a->wide - 1 + 31) / 32, g.n_heads), 256, 0, stream,
                       static_cast<const float*>(g.part), s.ld, s.splits, g.n_heads, h0, a->high, a->wide, by_position, a->heads,
                       a->buckets ? 0 : a->add);
    if (r) return r - 400;
    count += 2;
  }
  if (a->buckets) {
    r = launch_chained(bias_buckets_kernel, dim3(a->table_rows, (a->heads + 31) / 32), 256, 0, stream, *a,
                       static_cast<const float*>(by_position), p.off);
    if (r) return r - 500;
    ++count;
  }
  return count;
}
