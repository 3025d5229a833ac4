// shared_prefix.cuh -- what the kernels of the shared-prefix decode have in
// common: their parameters, the partial rows they leave in the workspace and
// the join of a row's partials.
#pragma once

#include "common.cuh"
#include "host_util.h"
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
// The prefix's parts for few rows, eight rows at a time.
int launch_shared_prefix_mma(const SharedParams& p, const b200_kv_pool_t& pool, int zero_count,
                             cudaStream_t stream);

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

// For own-key CTAs with nothing to join: what comes after the own-key kernel on
// the stream may take it that the prefix's kernel has ended too, so that the
// last CTA, whatever it does, ends after it.
__device__ __forceinline__ void end_after_previous() {
  if (blockIdx.x == gridDim.x - 1) wait_for_previous();
}

// Launches an own-key kernel, with leave to begin before the kernel ahead of it
// has ended where that is the prefix's.
template <typename... Params, typename... Args>
int launch_own(void (*kern)(Params...), int64_t grid, int block, int smem, cudaStream_t stream, bool overlap,
               const Args&... args) {
  if (grid > 0x7fffffffLL) return fail(B200_ERR_UNSUPPORTED, "shared prefix: grid too large");
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(static_cast<unsigned>(block));
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = overlap ? 1 : 0;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
  return e == cudaSuccess ? B200_OK : cuda_fail(e, "shared prefix own-key launch");
}

// The joined row (g, R), by one warp: sum_s 2^(m_s - M) acc_s / sum_s 2^(m_s -
// M) l_s over the prefix's slots and the first `parts` own ones (at most 96 in
// all).  A lane holds the factors of every 32nd part and four elements of the
// row; eight parts' loads are on their way together.
__device__ __forceinline__ void join_row(const SharedParams& p, int g, int R, int parts) {
  constexpr int kHeld = 3;
  const int lane = threadIdx.x & 31;
  const int64_t slot0 = (static_cast<int64_t>(g) * p.rows + R) * p.ns;
  const int n = p.np + parts;
  const float2* ml = reinterpret_cast<const float2*>(p.ml) + slot0;
  float2 v[kHeld];
  float M = -INFINITY, sum = 0.f, f[kHeld];
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    v[i] = lane + 32 * i < n ? __ldcg(ml + lane + 32 * i) : make_float2(-INFINITY, 0.f);
    M = fmaxf(M, v[i].x);
  }
#pragma unroll
  for (int w = 16; w >= 1; w >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, w));
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    // A part without a weight (no key, or a slot that stays unused) has no factor.
    f[i] = v[i].x == -INFINITY ? (v[i].y == 0.f ? 0.f : 1.f) : exp2f(v[i].x - M);
    sum = fmaf(f[i], v[i].y, sum);
  }
#pragma unroll
  for (int w = 16; w >= 1; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
  const float inv = 1.0f / sum;
  const bool mine = lane * 4 < p.D;
  const float* acc = p.acc + slot0 * p.D + lane * 4;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int j0 = 0; j0 < n; j0 += 8) {
    float4 x[8];
    float fj[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int j = j0 + k;
      fj[k] = __shfl_sync(0xffffffffu, j < 32 ? f[0] : j < 64 ? f[1] : f[2], j & 31) * inv;
      x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (j < n && fj[k] != 0.f && mine)
        x[k] = __ldcg(reinterpret_cast<const float4*>(acc + static_cast<int64_t>(j) * p.D));
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      a.x = fmaf(fj[k], x[k].x, a.x), a.y = fmaf(fj[k], x[k].y, a.y);
      a.z = fmaf(fj[k], x[k].z, a.z), a.w = fmaf(fj[k], x[k].w, a.w);
    }
  }
  if (!mine) return;
  const int b = R / p.rep, h = g * p.rep + R % p.rep;
  const int64_t at = b * p.os0 + h * p.os1 + lane * 4 * p.os2;
  store_elem(p.out, at, p.out_dtype, a.x);
  store_elem(p.out, at + p.os2, p.out_dtype, a.y);
  store_elem(p.out, at + 2 * p.os2, p.out_dtype, a.z);
  store_elem(p.out, at + 3 * p.os2, p.out_dtype, a.w);
}

}  // namespace b200
