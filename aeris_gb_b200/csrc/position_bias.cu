// Learned bias by relative position in window attention: what stands around the attention kernels (attention.cu), and the
// gradient of the table.
//
//   s_ij = scale q_i k_j + table[bucket(pos_i - pos_j), head], p = softmax_j(s), o = p v
//   ds = p (dp - delta), dp = dO v^T, delta = rowsum(p dp);  dtable[b, head] = sum of ds over windows and the pairs of bucket b
//
// The bias of a pair is a function of the difference of two tokens' places: with at(t) = y pitch + x it is entry
// at(i) - at(j) + at(last) of a table by relative position, which is all that the attention kernels read: one table of
// (2 high - 1) rows of `pitch` floats for a head, whatever the buckets, in log2 units, instead of an N x N matrix. The pitch is the
// least from 2 wide - 1 on that is `wide` more than a multiple of 32: from one token to the next `at` then grows by one
// modulo 32 even where a row of the window ends, and 32 queries read 32 banks of shared memory.
#include "common.cuh"
#include "api.h"
#include "host.h"
#include "cluster.cuh"
#include "position_bias.cuh"

namespace aeris {

namespace {

constexpr int PB_TILE = 128;

struct Place {
  int n;              // tokens of a window
  int pitch, zero;    // of the table's rows; entry of a token and itself
  int size;           // floats from one head's table to the next: whole vectors
  int at_words;       // `at`, up to the next multiple of 128 behind the window's end
};
Place place_of(int high, int wide) {
  Place p;
  p.n = high * wide;
  p.pitch = wide + (wide - 1 + 31) / 32 * 32;
  p.zero = (high - 1) * p.pitch + wide - 1;
  p.size = ((2 * high - 1) * p.pitch + 3) / 4 * 4;
  p.at_words = (p.n + 127) / 128 * 128;
  return p;
}
BiasSource source_of(const AerisBiasedAttn* a, const Place& p) {
  return {a->table, a->buckets, a->table_rows, a->heads, a->high, a->wide, p.pitch, a->table_bf16, a->buckets64, a->status};
}

// The tables by relative position [heads, size] in log2 units, and the places of the tokens.
__global__ void __launch_bounds__(256) bias_expand_kernel(const BiasSource s, float* out, int* at, const Place pl) {
  chain_point();
  const int i = blockIdx.x * 256 + threadIdx.x, head = blockIdx.y;
  if (i < pl.size) out[static_cast<long long>(head) * pl.size + i] = s.entry(i, head);
  if (head == 0 && i < pl.at_words) at[i] = s.at(i < pl.n ? i : pl.n - 1);
}

// ------------------------------------------------------------------------------------------ sums of dS over windows
// A tile is 128 queries x TK keys of one head, taken through all windows: S = Q K^T and dP = dO V^T of one window and the next
// into TMEM in turn, while p (dp - delta) of the one before is added up in registers. CTAs take whole tiles in rounds, all of them
// window after window at the same time, so that tiles of a head find their operands in L2 (runs of tiles that start in
// different windows, 128 x 256: 1.19 ms where rounds took 0.88). The windows of the tiles that are left for the last round are one sequence
// of steps, of which every CTA takes a run: no atomics, and no round of a few tiles. A tile whose last window is in a CTA's run is
// written to its place, what goes on in the next CTA's to `extra`, which bias_join_kernel adds.
//
// With p = 2^(c s + b - lse) the bias b of a pair is the same for all windows: 2^(c s - lse) (dp - delta) is added up and the sum
// multiplied by 2^b at the end, where every pair of a warp's is visible and |b| is at most 64 (a probability below 2^-62 may then be
// taken for zero); else b is added to every score.
//
// What bounds it is the operands' way from L2, 64 KB a window: loads and products alone take 0.62 of the 0.75 ms (72 windows of 30 x 30, 24
// heads of 64), 11 TB/s; the exponentials of a window take 1,024 cycles. Tiles of 128 x 256 read 48 KB for 128 x 128, but two
// windows' operands fill the shared memory then: 0.69 ms of loads alone, 0.88 in all.
template <int DCH> struct BgCfg {
  static constexpr int TK = DCH == 1 ? 128 : 64, CPT = TK / 4;
  static constexpr int QB = DCH * 16384, KB = DCH * TK * 128;
  static constexpr int NST = DCH == 1 ? 3 : 2, STAGE = 2 * QB + 2 * KB;      // ring of Q | dO | K | V
  // warps: math, loads, products, two without work; registers: together what 640 threads are launched with (96 each)
  static constexpr int MATH = 16, W_LOAD = MATH, W_MMA = MATH + 1, THREADS = 32 * (MATH + 4);
  static constexpr int REGS_MATH = 104, REGS_REST = 64, REGS = 32 * (MATH * REGS_MATH + 4 * REGS_REST);
  static constexpr int BARS = NST * STAGE, TMEM = 4 * TK, SMEM = BARS + 256 + 1024;
  static constexpr int TILE_FLOATS = PB_TILE * TK;
  static_assert(SMEM <= 227 * 1024, "shared memory");
};

struct BgParams {
  const float *lse, *delta, *table;
  const int* at;
  float *part, *extra;        // [heads at hand, n, ld]; [CTAs, 128, TK]
  long long ld;
  int n, heads, n_win, size, zero, head0, n_heads;
  float scale_log2;
  int* status;
};

__device__ __forceinline__ float bg_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct BgTile {
  int head, ti, tj;           // head: of those at hand
};
__device__ __forceinline__ BgTile bg_tile(int t, int n, int tm, int tk) {      // tiles of tm queries x tk keys
  const int nj = (n + tk - 1) / tk, ni = (n + tm - 1) / tm;
  BgTile b;
  const int r = t / nj;
  b.tj = t - r * nj;
  b.head = r / ni;
  b.ti = r - b.head * ni;
  return b;
}
// Who takes what: CTAs take `rounds` rounds of whole tiles, and the first `runs` of them runs of the steps (tile, window) that are left, as
// long as one another. runs = 0: what is left are whole tiles, one for a CTA.
struct BgPlan {
  int tiles, ctas, rounds, steps, runs;
  __host__ __device__ __forceinline__ int first(int b) const { return static_cast<int>(static_cast<long long>(steps) * b / runs); }
};
// What a CTA does, piece by piece: windows [w0, w1) of tile t.
struct BgWork {
  const BgPlan& p;
  int n_win, cta, round = 0, u = 0, u1 = 0, t = 0, w0 = 0, w1 = 0;
  __device__ __forceinline__ BgWork(const BgPlan& plan, int n_win_, int cta_) : p(plan), n_win(n_win_), cta(cta_) {
    if (cta < p.runs) {
      u = p.first(cta);
      u1 = p.first(cta + 1);
    }
  }
  __device__ __forceinline__ bool next() {
    const int whole = round * p.ctas + cta;
    if (round < p.rounds || (!p.runs && whole < p.tiles)) {
      ++round;
      t = whole;
      w0 = 0;
      w1 = n_win;
      return true;
    }
    if (u >= u1) return false;
    const int r = u / n_win;
    t = p.rounds * p.ctas + r;
    w0 = u - r * n_win;
    w1 = min(n_win, w0 + u1 - u);
    u += w1 - w0;
    return true;
  }
};

template <int DCH>
__global__ void __launch_bounds__(BgCfg<DCH>::THREADS, 1)
bias_grad_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_do,
                 const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const BgParams p,
                 const BgPlan plan) {
  using C = BgCfg<DCH>;
  constexpr int TK = C::TK, CPT = C::CPT, NST = C::NST;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::BARS);     // [NST]
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
  if (threadIdx.x == 0) {
    prefetch_tmap(&tm_q); prefetch_tmap(&tm_do); prefetch_tmap(&tm_k); prefetch_tmap(&tm_v);
    for (int i = 0; i < NST; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(&s_full[i], 1); mbar_init(&s_empty[i], C::MATH); }
    fence_barrier_init();
  }
  if (warp == C::W_MMA) { tmem_alloc(tmem_slot, C::TMEM); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  chain_point();

  if (warp >= C::MATH) regs_dec<C::REGS_REST>();
  if (warp == C::W_LOAD) {
    if (elect_one_sync()) {
      int st = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (BgWork k(plan, p.n_win, blockIdx.x); ok && k.next();) {
        const BgTile b = bg_tile(k.t, p.n, PB_TILE, TK);
        const int head = p.head0 + b.head;
        for (int w = k.w0; w < k.w1; ++w) {
          if (!mbar_wait_poll(&empty[st], ph ^ 1, p.status, ERR_TIMEOUT_ATTN)) { ok = false; break; }
          uint8_t* s = smem + st * C::STAGE;
          mbar_expect_tx(&full[st], C::STAGE);
#pragma unroll
          for (int c = 0; c < DCH; ++c) {
            tma_load_4d(s + c * 16384, &tm_q, &full[st], c * 64, head, b.ti * PB_TILE, w);
            tma_load_4d(s + 2 * C::QB + c * (TK * 128), &tm_k, &full[st], c * 64, head, b.tj * TK, w);
            tma_load_4d(s + C::QB + c * 16384, &tm_do, &full[st], c * 64, head, b.ti * PB_TILE, w);
            tma_load_4d(s + 2 * C::QB + C::KB + c * (TK * 128), &tm_v, &full[st], c * 64, head, b.tj * TK, w);
          }
          if (++st == NST) { st = 0; ph ^= 1; }
        }
      }
      for (int i = 0; i < NST && ok; ++i) {      // every stage has been released: no copy is under way at exit
        ok = mbar_wait_poll(&empty[st], ph ^ 1, p.status, ERR_TIMEOUT_ATTN);
        if (++st == NST) { st = 0; ph ^= 1; }
      }
    }
  } else if (warp == C::W_MMA) {
    if (elect_one_sync()) {
      constexpr uint32_t idesc = make_idesc_bf16(PB_TILE, TK, 0, 0);
      int st = 0, buf = 0;
      uint32_t ph = 0, b_ph = 0;
      bool ok = true;
      for (BgWork k(plan, p.n_win, blockIdx.x); ok && k.next();) {
        for (int w = k.w0; w < k.w1; ++w) {
          ok = mbar_wait_poll(&s_empty[buf], b_ph ^ 1, p.status, ERR_TIMEOUT_ATTN) &&
               mbar_wait_poll(&full[st], ph, p.status, ERR_TIMEOUT_ATTN);
          if (!ok) break;
          tc_fence_after();
          const uint32_t s = smem_u32(smem + st * C::STAGE), d = tmem_base + buf * 2 * TK;
#pragma unroll
          for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int kk = 0; kk < 4 * DCH; ++kk)
              umma_ss(d + m * TK, make_smem_desc(s + m * C::QB + (kk >> 2) * 16384 + (kk & 3) * 32, 0, 1024),
                      make_smem_desc(s + 2 * C::QB + m * C::KB + (kk >> 2) * (TK * 128) + (kk & 3) * 32, 0, 1024), idesc, kk > 0);
          tc_commit(&empty[st]);
          tc_commit(&s_full[buf]);
          if (++st == NST) { st = 0; ph ^= 1; }
          if (++buf == 2) { buf = 0; b_ph ^= 1; }
        }
      }
    }
  } else if (warp < C::MATH) {
    regs_inc<C::REGS_MATH>();
    const int q = warp & 3, g = warp >> 2;
    const uint32_t t0 = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + g * CPT;
    const uint64_t sl = f2_pack(p.scale_log2, p.scale_log2);
    const long long stat_step = static_cast<long long>(p.heads) * p.n;
    int buf = 0;
    uint32_t b_ph = 0;
    bool ok = true;
    for (BgWork work(plan, p.n_win, blockIdx.x); ok && work.next();) {
      const int w1 = work.w1;
      int w = work.w0;
      const BgTile b = bg_tile(work.t, p.n, PB_TILE, TK);
      const int row0 = b.ti * PB_TILE + q * 32, row = row0 + lane, col = b.tj * TK + g * CPT;
      const bool in = row < p.n, has = row0 < p.n && col < p.n;       // has: some of this warp's pairs are in the window
      const float* bias = p.table + static_cast<long long>(p.head0 + b.head) * p.size + p.zero + p.at[in ? row : p.n - 1];    // bias[-at[j]]
      uint64_t sum[CPT / 2];
      bool near = true;
#pragma unroll
      for (int i = 0; i < CPT / 2; ++i) sum[i] = 0ull;
      if (has)
#pragma unroll 4
        for (int i = 0; i < CPT; ++i) near = near && fabsf(bias[-p.at[min(col + i, p.n - 1)]]) <= 64.f;       // no NaN either
      near = __all_sync(0xffffffffu, near);
      const long long stat = static_cast<long long>(p.head0 + b.head) * p.n + (in ? row : p.n - 1);
      float lse = p.lse[stat + w * stat_step], delta = p.delta[stat + w * stat_step];
      // 16 columns from column c on
      auto add = [&](const uint32_t (&s)[16], const uint32_t (&dp)[16], uint64_t nl, uint64_t nd, int c, bool with_bias) {
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          uint64_t e = f2_fma(f2_pack(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), sl, nl);
          if (with_bias) {          // the places go on behind the window's end
            const int2 a = *reinterpret_cast<const int2*>(p.at + col + c + i);
            e = f2_add(e, f2_pack(bias[-a.x], bias[-a.y]));
          }
          float e0, e1;
          f2_unpack(e, e0, e1);
          const uint64_t d = f2_add(f2_pack(__uint_as_float(dp[i]), __uint_as_float(dp[i + 1])), nd);
          const int k = (c + i) / 2;
          sum[k] = f2_fma(f2_pack(bg_exp2(e0), bg_exp2(e1)), d, sum[k]);
        }
      };
      for (; w < w1; ++w) {
        const uint64_t nl = f2_pack(-lse, -lse), nd = f2_pack(-delta, -delta);
        if (w + 1 < w1) {
          lse = p.lse[stat + (w + 1) * stat_step];
          delta = p.delta[stat + (w + 1) * stat_step];
        }
        ok = mbar_wait_warp(&s_full[buf], b_ph, p.status, ERR_TIMEOUT_ATTN);
        if (!ok) break;
        tc_fence_after();
        if (has) {
          const uint32_t tS = t0 + buf * 2 * TK, tD = tS + TK;
#pragma unroll
          for (int c = 0; c < CPT; c += 16) {
            uint32_t s[16], dp[16];
            tmem_ld16(tS + c, s);
            tmem_ld16(tD + c, dp);
            tmem_wait_ld();
            if (c + 16 == CPT) {
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&s_empty[buf]);
            }
            if (near) add(s, dp, nl, nd, c, false);
            else if (col + c < p.n) add(s, dp, nl, nd, c, true);
          }
        } else {
          __syncwarp();
          if (lane == 0) mbar_arrive(&s_empty[buf]);
        }
        if (++buf == 2) { buf = 0; b_ph ^= 1; }
      }
      if (!ok || failed(p.status)) break;
      float* dst = w1 == p.n_win ? p.part + (static_cast<long long>(b.head) * p.n + row) * p.ld + col       // ld a multiple of 4
                                 : p.extra + static_cast<long long>(blockIdx.x) * C::TILE_FLOATS + (q * 32 + lane) * TK + g * CPT;
      if (has && in)
#pragma unroll
        for (int i = 0; i < CPT; i += 4)
          if (col + i < p.n) {
            float v[4];
            f2_unpack(sum[i / 2], v[0], v[1]);
            f2_unpack(sum[i / 2 + 1], v[2], v[3]);
            if (near) {
#pragma unroll
              for (int k = 0; k < 4; ++k) v[k] *= bg_exp2(bias[-p.at[min(col + i + k, p.n - 1)]]);
            }
            *reinterpret_cast<float4*>(dst + i) = make_float4(v[0], v[1], v[2], v[3]);
          }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == C::W_MMA) tmem_dealloc(tmem_base, C::TMEM);
}

// The same for more than 64 channels and 128 tokens, by pairs of CTAs (tcgen05.mma.cta_group::2): a tile is 256 queries, 128 of each
// CTA, x 128 keys, of which a CTA brings in half. A CTA then reads 96 KB from L2 for 128 x 128 pairs where one alone reads 192. 30 windows
// of 30 x 30, 24 heads of 128: 612 -> 456 us. With 64 channels (256 x 256, sums of 256 keys a row) the exponentials and the hand-over between
// CTAs take what the reads gave: 72 windows, 24 heads 777 us for 755, 100 windows of 16 x 16, 8 heads 206 for 188 (whole backward pass).
struct Bg2Cfg {
  static constexpr int TK = 128, CPT = 32, DCH = 2, QB = DCH * 16384, KB = DCH * 8192, NST = 2, STAGE = 2 * QB + 2 * KB;
  // warps and registers as above
  static constexpr int MATH = 16, W_LOAD = MATH, W_MMA = MATH + 1, THREADS = 32 * (MATH + 4);
  static constexpr int REGS_MATH = 104, REGS_REST = 64, REGS = 32 * (MATH * REGS_MATH + 4 * REGS_REST);
  static constexpr int BARS = NST * STAGE, SMEM = BARS + 256 + 1024, TILE_FLOATS = 2 * PB_TILE * TK;
  static_assert(SMEM <= 227 * 1024, "shared memory");
};

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Bg2Cfg::THREADS, 1)
bias_grad2_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_do,
                  const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const BgParams p,
                  const BgPlan plan) {
  using C = Bg2Cfg;
  constexpr int TK = C::TK, NST = C::NST, DCH = C::DCH, CPT = C::CPT;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::BARS);     // [NST], of the leader: both CTAs' copies
  uint64_t* empty = full + NST;
  uint64_t* s_full = empty + NST;       // [2]
  uint64_t* s_empty = s_full + 2;       // [2], of the leader: an arrival per warp of both CTAs
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(s_empty + 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_ctarank()), pair = blockIdx.x >> 1;
  __shared__ int s_abort;       // an earlier kernel has failed: the pair leaves, as its leader says
  if (threadIdx.x == 0) {
    s_abort = failed(p.status) ? 1 : 0;
    prefetch_tmap(&tm_q); prefetch_tmap(&tm_do); prefetch_tmap(&tm_k); prefetch_tmap(&tm_v);
    for (int i = 0; i < NST; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(&s_full[i], 1); mbar_init(&s_empty[i], 2 * C::MATH); }
    fence_barrier_init();
  }
  if (warp == C::W_MMA) { tmem_alloc2(tmem_slot, 512); tmem_relinquish2(); }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();       // both CTAs' barriers are initialised and tensor memory is allocated before anyone signals
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const bool gone = ld_shared_cluster_u32(map_to_cta(smem_u32(&s_abort), 0)) != 0;
  chain_point();

  if (!gone && warp >= C::MATH) regs_dec<C::REGS_REST>();
  if (gone) {
    // nothing is under way
  } else if (warp == C::W_LOAD) {
    if (elect_one_sync()) {
      int st = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (BgWork k(plan, p.n_win, pair); ok && k.next();) {
        const BgTile b = bg_tile(k.t, p.n, 2 * PB_TILE, TK);
        const int head = p.head0 + b.head, row0 = (2 * b.ti + rank) * PB_TILE, col0 = b.tj * TK + rank * 64;
        for (int w = k.w0; w < k.w1; ++w) {
          if (!mbar_wait_poll(&empty[st], ph ^ 1, p.status, ERR_TIMEOUT_ATTN)) { ok = false; break; }
          uint8_t* s = smem + st * C::STAGE;
          if (rank == 0) mbar_expect_tx(&full[st], 2 * C::STAGE);
          const uint32_t fb = map_to_cta(smem_u32(&full[st]), 0);
#pragma unroll
          for (int c = 0; c < DCH; ++c) {
            tma_load_4d_pair(s + c * 16384, &tm_q, fb, c * 64, head, row0, w);
            tma_load_4d_pair(s + 2 * C::QB + c * 8192, &tm_k, fb, c * 64, head, col0, w);
            tma_load_4d_pair(s + C::QB + c * 16384, &tm_do, fb, c * 64, head, row0, w);
            tma_load_4d_pair(s + 2 * C::QB + C::KB + c * 8192, &tm_v, fb, c * 64, head, col0, w);
          }
          if (++st == NST) { st = 0; ph ^= 1; }
        }
      }
      // after a time-out: the tiles that the issuer did not take, of both CTAs (a stage never filled counts as there)
      for (int s = 0; s < NST && !ok && rank == 0; ++s) {
        if (--st < 0) { st = NST - 1; ph ^= 1; }
        if (!mbar_wait_poll(&full[st], ph, nullptr, 0)) break;
      }
    }
  } else if (warp == C::W_MMA) {
    if (rank == 0 && elect_one_sync()) {
      constexpr uint32_t idesc = make_idesc_bf16(2 * PB_TILE, TK, 0, 0);
      int st = 0, buf = 0;
      uint32_t ph = 0, b_ph = 0;
      bool ok = true, any = false;
      for (BgWork k(plan, p.n_win, pair); ok && k.next();) {
        for (int w = k.w0; w < k.w1; ++w) {
          ok = mbar_wait_poll(&s_empty[buf], b_ph ^ 1, p.status, ERR_TIMEOUT_ATTN) &&
               mbar_wait_poll(&full[st], ph, p.status, ERR_TIMEOUT_ATTN);
          if (!ok) break;
          tc_fence_after();
          const uint32_t s = smem_u32(smem + st * C::STAGE), d = tmem_base + buf * 2 * TK;
#pragma unroll
          for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int kk = 0; kk < 4 * DCH; ++kk)
              umma2_ss(d + m * TK, make_smem_desc(s + m * C::QB + (kk >> 2) * 16384 + (kk & 3) * 32, 0, 1024),
                       make_smem_desc(s + 2 * C::QB + m * C::KB + (kk >> 2) * 8192 + (kk & 3) * 32, 0, 1024), idesc, kk > 0);
          tc_commit2_mc(&empty[st], 0x3);
          tc_commit2_mc(&s_full[buf], 0x3);
          any = true;
          if (++st == NST) { st = 0; ph ^= 1; }
          if (++buf == 2) { buf = 0; b_ph ^= 1; }
        }
      }
      // the last products have completed, whether those who wait for them gave up or not
      if (any) {
        if (--st < 0) { st = NST - 1; ph ^= 1; }
        mbar_wait_poll(&empty[st], ph, nullptr, 0);
      }
    }
  } else if (warp < C::MATH) {
    regs_inc<C::REGS_MATH>();
    const int q = warp & 3, g = warp >> 2;
    const uint32_t t0 = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + g * CPT;
    const uint64_t sl = f2_pack(p.scale_log2, p.scale_log2);
    const long long stat_step = static_cast<long long>(p.heads) * p.n;
    int buf = 0;
    uint32_t b_ph = 0;
    bool ok = true;
    for (BgWork work(plan, p.n_win, pair); ok && work.next();) {
      const int w1 = work.w1;
      int w = work.w0;
      const BgTile b = bg_tile(work.t, p.n, 2 * PB_TILE, TK);
      const int row0 = (2 * b.ti + rank) * PB_TILE + q * 32, row = row0 + lane, col = b.tj * TK + g * CPT;
      const bool in = row < p.n, has = row0 < p.n && col < p.n;
      const float* bias = p.table + static_cast<long long>(p.head0 + b.head) * p.size + p.zero + p.at[in ? row : p.n - 1];    // bias[-at[j]]
      uint64_t sum[CPT / 2];
      bool near = true;
#pragma unroll
      for (int i = 0; i < CPT / 2; ++i) sum[i] = 0ull;
      if (has)
#pragma unroll 4
        for (int i = 0; i < CPT; ++i) near = near && fabsf(bias[-p.at[min(col + i, p.n - 1)]]) <= 64.f;       // no NaN either
      near = __all_sync(0xffffffffu, near);
      const long long stat = static_cast<long long>(p.head0 + b.head) * p.n + (in ? row : p.n - 1);
      float lse = p.lse[stat + w * stat_step], delta = p.delta[stat + w * stat_step];
      // 16 columns from column c on; one branch for all of them keeps their exponentials together
      auto add = [&](const uint32_t (&s)[16], const uint32_t (&dp)[16], uint64_t nl, uint64_t nd, int c, bool with_bias) {
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          uint64_t e = f2_fma(f2_pack(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), sl, nl);
          if (with_bias) {          // the places go on behind the window's end
            const int2 a = *reinterpret_cast<const int2*>(p.at + col + c + i);
            e = f2_add(e, f2_pack(bias[-a.x], bias[-a.y]));
          }
          float e0, e1;
          f2_unpack(e, e0, e1);
          const uint64_t d = f2_add(f2_pack(__uint_as_float(dp[i]), __uint_as_float(dp[i + 1])), nd);
          sum[(c + i) / 2] = f2_fma(f2_pack(bg_exp2(e0), bg_exp2(e1)), d, sum[(c + i) / 2]);
        }
      };
      for (; w < w1; ++w) {
        const uint64_t nl = f2_pack(-lse, -lse), nd = f2_pack(-delta, -delta);
        if (w + 1 < w1) {
          lse = p.lse[stat + (w + 1) * stat_step];
          delta = p.delta[stat + (w + 1) * stat_step];
        }
        ok = mbar_wait_warp(&s_full[buf], b_ph, p.status, ERR_TIMEOUT_ATTN);
        if (!ok) break;
        tc_fence_after();
        const uint32_t tS = t0 + buf * 2 * TK, tD = tS + TK, freed = map_to_cta(smem_u32(&s_empty[buf]), 0);
        if (has) {
#pragma unroll
          for (int c = 0; c < CPT; c += 16) {
            uint32_t s[16], dp[16];
            tmem_ld16(tS + c, s);
            tmem_ld16(tD + c, dp);
            tmem_wait_ld();
            if (c + 16 == CPT) {
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive_remote_relaxed(freed);
            }
            if (near) add(s, dp, nl, nd, c, false);
            else if (col + c < p.n) add(s, dp, nl, nd, c, true);
          }
        } else {
          __syncwarp();
          if (lane == 0) mbar_arrive_remote_relaxed(freed);
        }
        if (++buf == 2) { buf = 0; b_ph ^= 1; }
      }
      if (!ok || failed(p.status)) break;
      float* dst = w1 == p.n_win ? p.part + (static_cast<long long>(b.head) * p.n + row) * p.ld + col       // ld a multiple of 4
                                 : p.extra + static_cast<long long>(pair) * C::TILE_FLOATS + (rank * PB_TILE + q * 32 + lane) * TK + g * CPT;
      if (has && in)
#pragma unroll
        for (int i = 0; i < CPT; i += 4)
          if (col + i < p.n) {
            float v[4];
            f2_unpack(sum[i / 2], v[0], v[1]);
            f2_unpack(sum[i / 2 + 1], v[2], v[3]);
            if (near) {
#pragma unroll
              for (int k = 0; k < 4; ++k) v[k] *= bg_exp2(bias[-p.at[min(col + i + k, p.n - 1)]]);
            }
            *reinterpret_cast<float4*>(dst + i) = make_float4(v[0], v[1], v[2], v[3]);
          }
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();       // nobody leaves while the pair may still touch its shared memory or tensor memory
  tc_fence_after();
  if (warp == C::W_MMA) tmem_dealloc2(tmem_base, 512);
}

// Tiles that several CTAs took part in: what those before the last one left in `extra`, in their order, eight sequences of them beside one
// another. Block (t, y): parts y, y + gridDim.y, .. (32 vectors of a row each) of the t-th tile of the runs.
__global__ void __launch_bounds__(256) bias_join_kernel(const BgParams p, const BgPlan plan, int tm, int tk) {
  __shared__ float4 part[8][32];
  chain_point();
  const int u0 = blockIdx.x * p.n_win, u1 = u0 + p.n_win, v = threadIdx.x & 31, k = threadIdx.x >> 5;
  int b0 = static_cast<int>(static_cast<long long>(u0) * plan.runs / plan.steps), b1;      // those with its first and its last step
  while (plan.first(b0 + 1) <= u0) ++b0;
  while (plan.first(b0) > u0) --b0;
  b1 = static_cast<int>(static_cast<long long>(u1 - 1) * plan.runs / plan.steps);
  while (plan.first(b1 + 1) < u1) ++b1;
  while (plan.first(b1) >= u1) --b1;
  if (b0 == b1) return;
  const BgTile b = bg_tile(plan.rounds * plan.ctas + blockIdx.x, p.n, tm, tk);
  const int vecs = (min(tk, p.n - b.tj * tk) + 3) / 4, groups = (vecs + 31) / 32, rows = min(tm, p.n - b.ti * tm);
  for (int item = blockIdx.y; item < rows * groups; item += gridDim.y) {
    const int r = item / groups, c = (item - r * groups) * 32 + v;
    const bool in = c < vecs;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    if (in)
#pragma unroll 4
      for (int i = b0 + k; i < b1; i += 8) {
        const float4 x = *(reinterpret_cast<const float4*>(p.extra + (static_cast<long long>(i) * tm + r) * tk) + c);
        s.x += x.x; s.y += x.y; s.z += x.z; s.w += x.w;
      }
    part[k][v] = s;
    __syncthreads();
    if (k == 0 && in) {
      float4* dst = reinterpret_cast<float4*>(p.part + (static_cast<long long>(b.head) * p.n + b.ti * tm + r) * p.ld + b.tj * tk) + c;
      s = *dst;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float4 x = part[i][v];
        s.x += x.x; s.y += x.y; s.z += x.z; s.w += x.w;
      }
      *dst = s;
    }
    __syncthreads();
  }
}

// Sums of the pairs of one relative position: a block has 32 positions of one difference in y (a lane each), its warps
// share the queries. Lanes read neighbouring keys of one query: 128 bytes a load.
__global__ void __launch_bounds__(256) bias_sums_kernel(const float* part, long long ld, int head0, int high, int wide, float* out,
                                                        int heads, int add) {
  __shared__ float part_sum[8][32];
  chain_point();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int dy = static_cast<int>(blockIdx.x) - (high - 1), k = blockIdx.y * 32 + lane, dx = k - (wide - 1), hl = blockIdx.z;
  const int n = high * wide, y0 = max(0, dy), y1 = min(high, high + dy);
  const int nx = min(8, wide), ny = 8 / nx;         // warps along x, y
  const long long down = static_cast<long long>(wide) * (ld + 1) * ny;
  float s = 0.f;
  if (warp < nx * ny)
    for (int xi = warp % nx; xi < wide; xi += nx) {
      const int xj = xi - dx, y = y0 + warp / nx;
      if (xj >= 0 && xj < wide) {
        const float* src = part + (static_cast<long long>(hl) * n + y * wide + xi) * ld + (y - dy) * wide + xj;
#pragma unroll 8
        for (int r = y; r < y1; r += ny, src += down) s += *src;
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

}  // namespace

}  // namespace aeris

#include "position_bias_small.cuh"

namespace aeris {

namespace {

constexpr long long PART_BYTES = 256ll << 20;

// How the sums of dS are taken: heads at a time (their matrices take at most 256 MB, or are one head's).
struct SumsPlan {
  int heads, tm, tk;
  bool pairs;
  long long ld, part, extra;      // bytes
};
SumsPlan plan_sums(int n_win, int n, int heads, int head_dim) {
  SumsPlan s;
  s.pairs = n > PB_TILE && head_dim > 64;      // see Bg2Cfg
  s.tm = s.pairs ? 2 * PB_TILE : PB_TILE;
  s.tk = s.pairs ? Bg2Cfg::TK : head_dim <= 64 ? BgCfg<1>::TK : BgCfg<2>::TK;
  s.ld = (n + 3) / 4 * 4;
  const long long one = 4ll * n * s.ld, tiles = static_cast<long long>((n + s.tm - 1) / s.tm) * ((n + s.tk - 1) / s.tk);
  s.heads = static_cast<int>(PART_BYTES / one);
  if (s.heads < 1) s.heads = 1;
  if (s.heads > heads) s.heads = heads;
  // tiles and steps are counted in 32 bits
  while (s.heads > 1 && tiles * s.heads * n_win > 0x3fffffff) s.heads /= 2;
  s.part = one * s.heads;
  s.extra = 4ll * num_sms() * PB_TILE * s.tk;
  return s;
}

// Runs of four steps at least, for a run costs about as much to start and to join; where tiles have few windows none.
BgPlan plan_tiles(int tiles, int n_win, int units) {
  BgPlan p{};
  p.tiles = tiles;
  const bool split = n_win > 16;
  const long long steps = static_cast<long long>(tiles) * n_win;
  p.ctas = split && tiles < units ? static_cast<int>((steps + 3) / 4 < units ? (steps + 3) / 4 : units) : (tiles < units ? tiles : units);
  p.rounds = tiles / p.ctas;
  const int left = tiles - p.rounds * p.ctas;
  if (split && left) {
    p.steps = left * n_win;
    p.runs = p.steps < p.ctas ? p.steps : p.ctas;
  }
  return p;
}

long long up(long long bytes) { return (bytes + 255) / 256 * 256; }

// Windows that position_bias_small.cuh takes; what it needs: sums by relative position of every run of windows, and where there are
// buckets those of all runs.
bool small(int high, int wide) { return static_cast<long long>(high) * wide <= SMALL_TOKENS; }
long long small_part(int n_win, int high, int wide, int heads, int head_dim) {
  return up(4ll * small_runs(n_win, high * wide, heads, head_dim, true) * heads * (2 * high - 1) * (2 * wide - 1));
}
SmallParams small_params(const AerisBiasedAttn* a, bool backward) {
  SmallParams p{};
  p.qkv = static_cast<const __nv_bfloat16*>(a->qkv); p.d_o = static_cast<const __nv_bfloat16*>(a->d_o);
  p.o = static_cast<__nv_bfloat16*>(a->o); p.dqkv = static_cast<__nv_bfloat16*>(a->dqkv); p.lse = a->lse;
  p.ld = a->ld_qkv; p.ldo = a->ld_o; p.ldg = a->ld_dqkv;
  p.n_win = a->n_win; p.n = a->high * a->wide; p.d = a->head_dim; p.scale = a->scale;
  p.runs = small_runs(a->n_win, p.n, a->heads, a->head_dim, backward);
  Place dense{};
  dense.pitch = 2 * a->wide - 1;
  p.source = source_of(a, dense);
  return p;
}
bool whole_rows(const void* p, long long ld) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % 8 == 0; }

struct Work {
  long long table, at, delta, rest, by_position, part, extra, total;
};
Work work_of(int n_win, int high, int wide, int heads, int head_dim, bool backward, bool with_table) {
  const Place p = place_of(high, wide);
  Work w{};
  const long long stats = 4ll * n_win * heads * p.n;
  w.at = up(4ll * heads * p.size);
  w.delta = w.at + up(4ll * p.at_words);
  w.rest = w.delta + (backward ? up(stats) : 0);
  w.by_position = w.rest + (backward ? up(4 * stats) : 0);
  w.part = w.by_position + (backward && with_table ? up(4ll * heads * (2 * high - 1) * (2 * wide - 1)) : 0);
  const SumsPlan s = plan_sums(n_win, p.n, heads, head_dim);
  w.extra = w.part + (backward && with_table ? up(s.part) : 0);
  w.total = w.extra + (backward && with_table ? up(s.extra) : 0);
  return w;
}

bool fits(const AerisBiasedAttn* a) {
  return a->n_win > 0 && a->high > 0 && a->wide > 0 && a->heads > 0 && a->head_dim > 0 && a->n_win <= 65535 && a->heads <= 65535 &&
         a->high <= 32768 && a->wide <= 32768 && static_cast<long long>(a->high) * a->wide <= 32768 && a->table && a->table_rows > 0 &&
         (reinterpret_cast<uintptr_t>(a->work) & 255) == 0 && a->ld_qkv <= 0x7fffffff && a->ld_o <= 0x7fffffff &&
         a->ld_dqkv <= 0x7fffffff;
}

int expand(const BiasSource& s, const Place& p, float* table, int* at, cudaStream_t stream) {
  const int most = p.size > p.at_words ? p.size : p.at_words;
  return launch_chained(bias_expand_kernel, dim3((most + 255) / 256, s.heads), 256, 0, stream, s, table, at, p);
}

template <int DCH>
int launch_bias_grad(const CUtensorMap (&m)[4], const BgParams& p, const BgPlan& plan, cudaStream_t stream, int& kernels) {
  static std::atomic<uint64_t> done{0};
  using C = BgCfg<DCH>;
  if (!once_a_device(done, [&] {
        // warpgroups that ask for more registers than the launch holds would wait for ever
        cudaFuncAttributes f;
        return cudaFuncSetAttribute(bias_grad_kernel<DCH>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) == cudaSuccess &&
               cudaFuncGetAttributes(&f, bias_grad_kernel<DCH>) == cudaSuccess && f.numRegs * C::THREADS >= C::REGS;
      }))
    return -20;
  ++kernels;
  return launch_chained(bias_grad_kernel<DCH>, plan.ctas, C::THREADS, C::SMEM, stream, m[0], m[1], m[2], m[3], p, plan);
}
// As many pairs as the device holds at once (a group of SMs with an odd number of them has one left over).
int pairs_held() {
  static std::atomic<uint64_t> done{0};
  static std::atomic<int> held{0};
  using C = Bg2Cfg;
  if (!once_a_device(done, [&] {        // see launch_bias_grad
        cudaFuncAttributes f;
        return cudaFuncSetAttribute(bias_grad2_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) == cudaSuccess &&
               cudaFuncGetAttributes(&f, bias_grad2_kernel) == cudaSuccess && f.numRegs * C::THREADS >= C::REGS;
      }))
    return 0;
  int pairs = held.load(std::memory_order_relaxed);
  if (!pairs) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(num_sms() / 2 * 2);
    cfg.blockDim = dim3(C::THREADS);
    cfg.dynamicSmemBytes = C::SMEM;
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim = {2, 1, 1};
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&pairs, bias_grad2_kernel, &cfg) != cudaSuccess || pairs <= 0 || pairs > num_sms() / 2)
      pairs = num_sms() / 2;
    held.store(pairs, std::memory_order_relaxed);
  }
  return pairs;
}
int launch_bias_grad2(const CUtensorMap (&m)[4], const BgParams& p, const BgPlan& plan, cudaStream_t stream, int& kernels) {
  using C = Bg2Cfg;
  ++kernels;
  return launch_chained(bias_grad2_kernel, 2 * plan.ctas, C::THREADS, C::SMEM, stream, m[0], m[1], m[2], m[3], p, plan);
}

}  // namespace

}  // namespace aeris

using namespace aeris;

extern "C" long long aeris_biased_attn_work_bytes(int n_win, int high, int wide, int heads, int head_dim, int backward, int with_table) {
  if (n_win <= 0 || high <= 0 || wide <= 0 || heads <= 0 || head_dim <= 0 || static_cast<long long>(high) * wide > 32768) return -1;
  if (small(high, wide)) {
    if (!backward || !with_table) return 0;
    return small_part(n_win, high, wide, heads, head_dim) + up(4ll * heads * (2 * high - 1) * (2 * wide - 1));
  }
  if (!backward) {
    BiasSource s{};
    s.high = high; s.wide = wide; s.pitch = place_of(high, wide).pitch;
    if (biased_fwd_reads_source(n_win, heads, head_dim, s)) return 0;
  }
  return work_of(n_win, high, wide, heads, head_dim, backward, with_table).total;
}

extern "C" int aeris_biased_attn_fwd(const AerisBiasedAttn* a, void* stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (!fits(a)) return -1;
  if (small(a->high, a->wide)) {
    if (a->head_dim > 128 || a->head_dim % 8 || !whole_rows(a->qkv, a->ld_qkv) || !whole_rows(a->o, a->ld_o) || !a->lse) return -3;
    const int r = launch_small(small_params(a, false), false, stream);
    return r ? r : 1;
  }
  const Place p = place_of(a->high, a->wide);
  const BiasSource source = source_of(a, p);
  if (biased_fwd_reads_source(a->n_win, a->heads, a->head_dim, source)) {
    const int r = attn_fwd_biased(a->qkv, static_cast<int>(a->ld_qkv), a->o, static_cast<int>(a->ld_o), a->lse, a->n_win, a->heads,
                                  a->head_dim, a->scale, source, nullptr, nullptr, p.size, stream);
    return r ? r - 100 : 1;
  }
  const Work w = work_of(a->n_win, a->high, a->wide, a->heads, a->head_dim, false, false);
  if (!a->work || a->work_bytes < w.total) return -2;
  uint8_t* work = static_cast<uint8_t*>(a->work);
  float* table = reinterpret_cast<float*>(work + w.table);
  int* at = reinterpret_cast<int*>(work + w.at);
  int r = expand(source, p, table, at, stream);
  if (r) return r;
  r = attn_fwd_biased(a->qkv, static_cast<int>(a->ld_qkv), a->o, static_cast<int>(a->ld_o), a->lse, a->n_win, a->heads, a->head_dim,
                      a->scale, source, table, at, p.size, stream);
  return r ? r - 100 : 2;
}

extern "C" int aeris_biased_attn_bwd(const AerisBiasedAttn* a, void* stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (!fits(a) || !a->d_o || !a->dqkv || !a->lse) return -1;
  const bool sums = a->dtable != nullptr;
  if (small(a->high, a->wide)) {
    const int size = (2 * a->high - 1) * (2 * a->wide - 1) * a->heads;
    const long long part = small_part(a->n_win, a->high, a->wide, a->heads, a->head_dim);
    if (a->head_dim > 128 || a->head_dim % 8 || !whole_rows(a->qkv, a->ld_qkv) || !whole_rows(a->d_o, a->ld_o) ||
        !whole_rows(a->dqkv, a->ld_dqkv))
      return -3;
    if (sums && (!a->work || a->work_bytes < part + up(4ll * size))) return -2;
    SmallParams s = small_params(a, true);
    if (sums) s.part = static_cast<float*>(a->work);
    int r = launch_small(s, true, stream);
    if (r || !sums) return r ? r : 1;
    float* out = a->buckets ? reinterpret_cast<float*>(static_cast<uint8_t*>(a->work) + part) : a->dtable;
    r = launch_chained(small_join_kernel, (size + 31) / 32, 256, 0, stream, static_cast<const float*>(s.part), out, s.runs, size,
                       a->buckets ? 0 : a->add);
    if (r || !a->buckets) return r ? r - 100 : 2;
    r = launch_chained(bias_buckets_kernel, dim3(a->table_rows, (a->heads + 31) / 32), 256, 0, stream, *a, static_cast<const float*>(out),
                       (2 * a->high - 1) * (2 * a->wide - 1));
    return r ? r - 500 : 3;
  }
  const Work w = work_of(a->n_win, a->high, a->wide, a->heads, a->head_dim, true, sums);
  if (!a->work || a->work_bytes < w.total) return -2;
  const Place p = place_of(a->high, a->wide);
  const BiasSource source = source_of(a, p);
  uint8_t* work = static_cast<uint8_t*>(a->work);
  float* table = reinterpret_cast<float*>(work + w.table);
  int* at = reinterpret_cast<int*>(work + w.at);
  float* delta = reinterpret_cast<float*>(work + w.delta);
  int r = expand(source, p, table, at, stream);
  if (r) return r;
  r = attn_bwd_biased(a->qkv, static_cast<int>(a->ld_qkv), a->o, a->d_o, static_cast<int>(a->ld_o), a->lse, delta,
                      reinterpret_cast<float*>(work + w.rest), a->dqkv, static_cast<int>(a->ld_dqkv), a->n_win, a->heads,
                      a->head_dim, a->scale, source, table, at, p.size, stream);
  if (r) return r - 100;
  int count = 4;
  if (!sums) return count;
  const int dch = a->head_dim <= 64 ? 1 : 2, hd = a->heads * a->head_dim;
  const SumsPlan s = plan_sums(a->n_win, p.n, a->heads, a->head_dim);
  const uint32_t keys = s.pairs ? 64 : s.tk;        // rows of K and V at a time
  const int units = s.pairs ? pairs_held() : num_sms();
  if (!units) return -20;
  const __nv_bfloat16* b = static_cast<const __nv_bfloat16*>(a->qkv);
  CUtensorMap m[4];
  const struct { const void* base; long long ld; uint32_t rows; } ops[4] = {
      {b, a->ld_qkv, PB_TILE}, {a->d_o, a->ld_o, PB_TILE}, {b + hd, a->ld_qkv, keys}, {b + 2 * hd, a->ld_qkv, keys}};
  for (int i = 0; i < 4; ++i)
    if ((r = make_tmap_heads_bf16(&m[i], ops[i].base, a->head_dim, a->heads, p.n, a->n_win, ops[i].ld, ops[i].rows))) return r - 200;
  BgParams g{};
  g.lse = a->lse; g.delta = delta; g.table = table; g.at = at; g.part = reinterpret_cast<float*>(work + w.part);
  g.extra = reinterpret_cast<float*>(work + w.extra); g.ld = s.ld;
  g.n = p.n; g.heads = a->heads; g.n_win = a->n_win; g.size = p.size; g.zero = p.zero;
  g.scale_log2 = a->scale * 1.4426950408889634f; g.status = a->status;
  float* by_position = a->buckets ? reinterpret_cast<float*>(work + w.by_position) : a->dtable;
  for (int h0 = 0; h0 < a->heads; h0 += s.heads) {
    g.head0 = h0;
    g.n_heads = a->heads - h0 < s.heads ? a->heads - h0 : s.heads;
    const BgPlan plan = plan_tiles((p.n + s.tm - 1) / s.tm * ((p.n + s.tk - 1) / s.tk) * g.n_heads, a->n_win, units);
    r = s.pairs ? launch_bias_grad2(m, g, plan, stream, count)
                : (dch == 1 ? launch_bias_grad<1>(m, g, plan, stream, count) : launch_bias_grad<2>(m, g, plan, stream, count));
    if (r) return r - 300;
    if (plan.runs) {
      const int tiles = plan.tiles - plan.rounds * plan.ctas;
      if ((r = launch_chained(bias_join_kernel, dim3(tiles, tiles < 32 ? 128 : 32), 256, 0, stream, g, plan, s.tm, s.tk))) return r - 300;
      ++count;
    }
    r = launch_chained(bias_sums_kernel, dim3(2 * a->high - 1, (2 * a->wide - 1 + 31) / 32, g.n_heads), 256, 0, stream,
                       static_cast<const float*>(g.part), s.ld, h0, a->high, a->wide, by_position, a->heads, a->buckets ? 0 : a->add);
    if (r) return r - 400;
    ++count;
  }
  if (a->buckets) {
    r = launch_chained(bias_buckets_kernel, dim3(a->table_rows, (a->heads + 31) / 32), 256, 0, stream, *a,
                       static_cast<const float*>(by_position), (2 * a->high - 1) * (2 * a->wide - 1));
    if (r) return r - 500;
    ++count;
  }
  return count;
}
