// The learned bias by relative position as the kernels see it, shared by position_bias.cu and attention.cu.
#pragma once
#include "common.cuh"
#include "api.h"

namespace aeris {

constexpr float BIAS_HIDDEN = -1e30f;      // entries of the learned table that are no larger hide the pairs of their bucket

// The learned table [rows, heads] behind the buckets of relative positions, windows of high x wide tokens. By relative position it is
// laid out in 2 high - 1 rows of `pitch` entries, of which 2 wide - 1 are used (see position_bias.cu).
struct BiasSource {
  const void *table, *buckets;
  int rows, heads, high, wide, pitch;
  int bf16, long_buckets;
  int* status;

  // Place of a token; entry at(i) - at(j) + at(last) is that of query i and key j.
  __host__ __device__ __forceinline__ int at(int t) const {
    const int y = t / wide;
    return y * pitch + t - y * wide;
  }
  // Entry k of head `head` in log2 units; -infinity hides. A bucket outside the table is recorded and hides.
  __device__ __forceinline__ float entry(int k, int head) const {
    const int r = k / pitch, c = k - r * pitch;
    if (r >= 2 * high - 1 || c >= 2 * wide - 1) return 0.f;       // between the rows: not read
    const int i = r * (2 * wide - 1) + c;
    long long b = i;
    if (buckets) b = long_buckets ? static_cast<const long long*>(buckets)[i] : static_cast<const int*>(buckets)[i];
    if (b < 0 || b >= rows) {
      if (status) atomicCAS(status, 0, ERR_BOUNDS);
      return -INFINITY;
    }
    const long long e = b * heads + head;
    const float v = bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(table)[e]) : static_cast<const float*>(table)[e];
    return v <= BIAS_HIDDEN ? -INFINITY : v * 1.4426950408889634f;
  }
};

// Forward with scores biased by relative position (attention.cu): fused qkv rows as aeris_attn_fwd, q in the first columns. `table`
// [heads, size] and `at`: what bias_expand_kernel writes, or null where biased_fwd_reads_source said so.
int attn_fwd_biased(const void* qkv, int ld, void* o, int ldo, float* lse, int n_win, int H, int head_dim, float scale,
                    const BiasSource& source, const float* table, const int* at, int size, void* stream);
bool biased_fwd_reads_source(int n_win, int H, int head_dim, const BiasSource& source);
// Backward. delta, rest: scratch of one and four floats per (window, head, token); delta holds dO . O afterwards, exact but for
// fp32 roundings.
int attn_bwd_biased(const void* qkv, int ldq, const void* o, const void* d_o, int ldo, const float* lse, float* delta, float* rest,
                    void* dqkv, int ldg, int n_win, int H, int head_dim, float scale, const BiasSource& source, const float* table,
                    const int* at, int size, void* stream);

}  // namespace aeris
