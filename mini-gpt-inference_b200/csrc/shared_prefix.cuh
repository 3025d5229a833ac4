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

// The most parts of a row: of the prefix and of its own keys.
constexpr int kPrefixParts = 64, kOwnParts = 32;

// Own keys and join, bf16 pool, kOwnRows rows of a key head to a CTA.  (16 rows
// take twice the registers and a longer code that has to be fetched first: 16
// query heads to each of 4 key heads, 64 sequences behind 4096 keys 45 us, two
// CTAs of eight rows 37 us.)  `overlap`: the kernel ahead on the stream is the
// prefix's.
constexpr int kOwnRows = 8;
int launch_shared_own_mma(const SharedParams& p, const b200_kv_pool_t& pool, bool overlap,
                          cudaStream_t stream);
// The prefix's parts, eight rows at a time.
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

// Two floats as bf16 rounded towards zero (their upper halves).  Where several
// bf16 pieces add up to a number, all but the last are chopped like this: what is
// left then has the number's sign, and kKeepSign of the number, less than f32
// itself rounds off, keeps it from being zero, so that every piece times an
// infinity is the same infinity.  (Pieces rounded to nearest leave rests of
// either sign or none: inf - inf, 0 * inf.)
constexpr float kKeepSign = 0x1p-30f;
__device__ __forceinline__ uint32_t chop_bf16(float lo, float hi) {
  return __byte_perm(__float_as_uint(lo), __float_as_uint(hi), 0x7632);
}

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

// The joined rows row0 .. row0 + nrows - 1 (at most 8) of key head g, by a block
// of 128 threads: sum_s 2^(m_s - M) acc_s / sum_s 2^(m_s - M) l_s over the
// prefix's slots and the first `parts` own ones.  `sm`:
// kJoinFloats of shared memory that the block is done with.  Four elements of a
// row are a thread's, or, where the rows are short or few, several threads' that
// share the parts out; the first loads are on their way before the factors are
// known.
constexpr int kJoinParts = kPrefixParts + kOwnParts, kJoinAhead = 8;
static_assert(kJoinParts % 32 == 0, "a lane's parts");
constexpr int kJoinFloats = 8 * kJoinParts + 128 * 4;
__device__ __forceinline__ void join_rows(const SharedParams& p, int g, int row0, int nrows, int parts,
                                          float* sm) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n = p.np + parts, quads = p.D / 4, items = nrows * quads;
  const int sharers = max(1, 128 / items);
  const int first = tid / items;  // of this thread's parts (sharers > 1)
  const int64_t slot0 = (static_cast<int64_t>(g) * p.rows + row0) * p.ns;
  float4 v[kJoinAhead];
  auto fetch = [&](int i, int j0) {
    const float* acc = p.acc + (slot0 + static_cast<int64_t>(i / quads) * p.ns + j0) * p.D + (i % quads) * 4;
#pragma unroll
    for (int k = 0; k < kJoinAhead; ++k)
      if (j0 + k * sharers < n)
        v[k] = __ldcg(reinterpret_cast<const float4*>(acc + static_cast<int64_t>(k * sharers) * p.D));
  };
  const int item0 = sharers > 1 ? tid % items : tid;
  const bool works = sharers > 1 ? first < sharers : tid < items;
  const int part0 = sharers > 1 ? first : 0;
  if (works) fetch(item0, part0);
  for (int r = warp; r < nrows; r += 4) {  // factors, a warp per row
    const float2* ml = reinterpret_cast<const float2*>(p.ml) + slot0 + static_cast<int64_t>(r) * p.ns;
    float2 x[kJoinParts / 32];
    float M = -INFINITY, sum = 0.f;
#pragma unroll
    for (int i = 0; i < kJoinParts / 32; ++i) {
      x[i] = lane + 32 * i < n ? __ldcg(ml + lane + 32 * i) : make_float2(-INFINITY, 0.f);
      M = fmaxf(M, x[i].x);
    }
#pragma unroll
    for (int w = 16; w >= 1; w >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, w));
#pragma unroll
    for (int i = 0; i < kJoinParts / 32; ++i) {
      // A part without a weight (no key, or a slot that stays unused) has no factor.
      const float f = x[i].x == -INFINITY ? (x[i].y == 0.f ? 0.f : 1.f) : exp2f(x[i].x - M);
      sum = fmaf(f, x[i].y, sum);
      x[i].x = f;
    }
#pragma unroll
    for (int w = 16; w >= 1; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
    const float inv = 1.0f / sum;
#pragma unroll
    for (int i = 0; i < kJoinParts / 32; ++i) sm[r * kJoinParts + lane + 32 * i] = x[i].x * inv;
  }
  __syncthreads();
  auto store = [&](int i, const float4& a) {
    const int R = row0 + i / quads, b = R / p.rep, h = g * p.rep + R % p.rep;
    const int64_t at = b * p.os0 + h * p.os1 + (i % quads) * 4 * p.os2;
    store_elem(p.out, at, p.out_dtype, a.x);
    store_elem(p.out, at + p.os2, p.out_dtype, a.y);
    store_elem(p.out, at + 2 * p.os2, p.out_dtype, a.z);
    store_elem(p.out, at + 3 * p.os2, p.out_dtype, a.w);
  };
  float4* share = reinterpret_cast<float4*>(sm + 8 * kJoinParts);
  if (works)
    for (int i = item0; i < items; i += sharers > 1 ? items : 128) {
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int j0 = part0; j0 < n; j0 += kJoinAhead * sharers) {
        if (i != item0 || j0 != part0) fetch(i, j0);
#pragma unroll
        for (int k = 0; k < kJoinAhead; ++k) {
          const int j = j0 + k * sharers;
          const float f = j < n ? sm[i / quads * kJoinParts + j] : 0.f;
          if (f == 0.f) continue;  // an unused slot holds anything
          a.x = fmaf(f, v[k].x, a.x), a.y = fmaf(f, v[k].y, a.y);
          a.z = fmaf(f, v[k].z, a.z), a.w = fmaf(f, v[k].w, a.w);
        }
      }
      if (sharers > 1)
        share[tid] = a;
      else
        store(i, a);
    }
  if (sharers == 1) return;
  __syncthreads();
  if (tid < items) {
    float4 a = share[tid];
    for (int k = 1; k < sharers; ++k) {
      const float4 x = share[tid + k * items];
      a.x += x.x, a.y += x.y, a.z += x.z, a.w += x.w;
    }
    store(tid, a);
  }
}

}  // namespace b200
