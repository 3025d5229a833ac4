// shared_prefix.cuh -- what the kernels of the shared-prefix decode have in
// common: their parameters, the partial rows they leave in the workspace and
// the join of a row's partials.
#pragma once

#include "common.cuh"
#include "kernels.h"

namespace b200 {

// Query head h of sequence b reads key/value head g = h / rep; row
// R = b * rep + h % rep of head g.  A row's softmax over the prefix and the
// sequence's own keys is computed in parts, each an unnormalised
//   acc = sum_j 2^(s_j - m) v_j,   m = max_j s_j,   l = sum_j 2^(s_j - m)
// with s = q.k log2(e) / sqrt(D): slots [0, np) of a row hold the prefix's
// parts, slots [np, ns) those of its own keys.
struct SharedParams {
  const void* q;
  void* out;
  int64_t qs0, qs1, qs2, os0, os1, os2;
  const void* k_pool;
  const void* v_pool;
  int64_t P, S;
  int64_t layer_row0;  // layer * P * S
  const void* prefix_table;
  int64_t pt_stride;
  const void* tables;
  int64_t ts0, ts1;
  int64_t table_width;
  const void* lens;
  int64_t len_stride;
  float* acc;    // [Hkv][rows][ns][D]
  float* ml;     // [Hkv][rows][ns][2]
  int32_t* cnt;  // [units of own keys], zero before the launch
  int32_t* status;
  int64_t prefix;
  int32_t B, Hq, Hkv, D, rep, rows;  // rows = B * rep
  int32_t s_shift;                   // log2(S)
  int32_t np, ns;
  int32_t prefix_per;   // keys of one prefix part (element kernels)
  int32_t own_splits;   // most parts of a sequence's own keys: ns - np
  int32_t own_min;      // fewest keys of such a part, unless it is the only one
  int32_t row_chunks;   // chunks of a key head's rep rows
  int32_t q_dtype, out_dtype;
  int32_t pt_i64, tables_i64, lens_i64;
  float qscale;  // log2(e) / sqrt(D)
};

// Own keys and join, bf16 pool and queries; the rows of a key head one CTA
// takes.  `overlap`: the kernel ahead on the stream is the prefix's.
int launch_shared_own_mma(const SharedParams& p, const b200_kv_pool_t& pool, bool overlap,
                          cudaStream_t stream);
int shared_own_rows(int64_t rep);

// The prefix on tensor cores: how its key tiles are cut.
struct TcSplit {
  int64_t units;   // up to 256 rows of a key head each
  int unit_tiles;  // key tiles of one unit
  int unit_pairs;  // units per key head
  int ctas;
  int np;          // most CTAs that share a unit
};
TcSplit shared_tc_split(int64_t rows, int64_t Hkv, int64_t prefix, int num_sms);
int launch_shared_prefix_tc(const SharedParams& s, const b200_kv_pool_t& pool, const TcSplit& t,
                            int zero_count, cudaStream_t stream);

// Keys [*k0, *k1) of part `split` of a sequence with n own keys; returns the
// number of parts (at least 1, also for n = 0).
__device__ __forceinline__ int own_range(const SharedParams& p, int64_t n, int split, int64_t* k0,
                                         int64_t* k1) {
  int64_t per = (n + p.own_splits - 1) / p.own_splits;
  per = max((per + 31) & ~int64_t(31), static_cast<int64_t>(p.own_min));
  const int parts = n > 0 ? static_cast<int>((n + per - 1) / per) : 1;
  *k0 = min(split * per, n);
  *k1 = min(*k0 + per, n);
  return parts;
}

// The own-key kernel may begin while the prefix's is still running:
// `let_next_start` allows it, `wait_for_previous` waits until the kernel ahead
// on the stream has ended and its writes can be read.
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// The joined row (g, R): element d of sum_s 2^(m_s - M) acc_s / sum_s
// 2^(m_s - M) l_s over the prefix's slots and the first `parts` own ones,
// for the elements of this thread (d = t, t + nt, ...).
__device__ __forceinline__ void join_row(const SharedParams& p, int g, int R, int parts, int t,
                                         int nt) {
  const int64_t slot0 = (static_cast<int64_t>(g) * p.rows + R) * p.ns;
  const int n = p.np + parts;
  float M = -INFINITY;
  for (int s = 0; s < n; ++s) M = fmaxf(M, __ldcg(&p.ml[(slot0 + s) * 2]));
  float L = 0.f;
  for (int s = 0; s < n; ++s) {
    const float m = __ldcg(&p.ml[(slot0 + s) * 2]);
    if (m != -INFINITY) L = fmaf(exp2f(m - M), __ldcg(&p.ml[(slot0 + s) * 2 + 1]), L);
  }
  const float inv = 1.0f / L;
  const int b = R / p.rep, h = g * p.rep + R % p.rep;
  for (int d = t; d < p.D; d += nt) {
    float o = 0.f;
    for (int s = 0; s < n; ++s) {
      const float m = __ldcg(&p.ml[(slot0 + s) * 2]);
      if (m != -INFINITY) o = fmaf(exp2f(m - M), __ldcg(&p.acc[(slot0 + s) * p.D + d]), o);
    }
    store_elem(p.out, b * p.os0 + h * p.os1 + d * p.os2, p.out_dtype, o * inv);
  }
}

}  // namespace b200
