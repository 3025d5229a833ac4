// shared_prefix.cu -- paged decode attention of a batch whose sequences share
// a prefix: the prefix's keys and values are read once for the whole batch.
//
//   out[b, h] = sum_j softmax_j(q[b, h].k_j / sqrt(D)) v_j
// over the prefix's keys (prefix_table) and the sequence's own (positions
// prefix .. context_length - 1 of its block table).  The softmax splits: the
// prefix's part is one product of all B * rep query rows of a key head with
// the prefix (arithmetic grows with the batch, bytes do not); the own parts
// are a matrix-vector product per sequence; parts are joined by their running
// maximum and sum.
//
// Element kernels (any pool and query type in f32; f32 pools, and pages of fewer
// than 8 tokens): a tile of R query
// rows in shared memory, key tiles of 32, thread tiles of scores and outputs
// in registers, online softmax in the log2 domain.
#include <math.h>
#include <stdio.h>

#include <algorithm>
#include <atomic>

#include "common.cuh"
#include "host_util.h"
#include "kernels.h"
#include "shared_prefix.cuh"

namespace b200 {
namespace {

constexpr int kKeys = 32;  // keys per tile of the element kernels

// Thread tile: TR x TC threads, RT rows and kKeys / TC keys (then DP / TC
// output columns, in float4 groups) each.
template <int R>
struct ElemTile;
template <>
struct ElemTile<64> {
  static constexpr int RT = 4, TC = 8;  // 16 x 8 threads
};
template <>
struct ElemTile<16> {
  static constexpr int RT = 1, TC = 8;  // 16 x 8 threads
};
template <>
struct ElemTile<8> {
  static constexpr int RT = 1, TC = 16;  // 8 x 16 threads
};

template <int R, int DP>
struct ElemSmem {
  static constexpr int LD = DP + 4;  // row pitch: float4 reads of 8 rows spread over the banks
  static constexpr int Q = 0, K = Q + R * LD, V = K + kKeys * LD, P = V + kKeys * LD;
  static constexpr int LP = kKeys + 1;
  static constexpr int ROWS = P + R * LP;  // int [2][kKeys]: pool rows of the next tiles' keys
  static constexpr int BYTES = (ROWS + 2 * kKeys) * 4;
};

// One part: R rows (row i of the tile is query row row0 + i of key head g,
// those from nrows on are empty) over keys [k0, k1) of a page list.
template <typename KV, int R, int DP>
struct ElemAttend {
  using T = ElemTile<R>;
  using L = ElemSmem<R, DP>;
  static constexpr int RT = T::RT, TC = T::TC, KPT = kKeys / TC;
  static constexpr int NG = (DP / 4 + TC - 1) / TC;  // float4 column groups per thread
  float m[RT], l[RT];
  float4 o[RT][NG];

  __device__ void run(const SharedParams& p, float* sm, int g, int row0, int nrows, int64_t k0,
                      int64_t k1, const void* table, int64_t tstride, int ti64, int64_t tlen) {
    const int tid = threadIdx.x;
    const int tr = tid / TC, tc = tid % TC;
    float* Q = sm + L::Q;
    float* K = sm + L::K;
    float* V = sm + L::V;
    float* Pm = sm + L::P;
    for (int i = tid; i < R * DP; i += 128) {
      const int r = i / DP, d = i % DP;
      float x = 0.f;
      if (r < nrows && d < p.D) {
        const int row = row0 + r;
        x = load_elem(p.q, (row / p.rep) * p.qs0 + (g * p.rep + row % p.rep) * p.qs1 + d * p.qs2,
                      p.q_dtype) * p.qscale;
      }
      Q[r * L::LD + d] = x;
    }
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      m[i] = -INFINITY;
      l[i] = 0.f;
#pragma unroll
      for (int c = 0; c < NG; ++c) o[i][c] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    const KV* kp = static_cast<const KV*>(p.k_pool);
    const KV* vp = static_cast<const KV*>(p.v_pool);
    constexpr int E = 16 / sizeof(KV);     // elements per 16-byte chunk
    constexpr int CH = DP / E;             // chunks per row
    constexpr int IT = kKeys * CH / 128;   // chunks of K (and of V) per thread and tile
    static_assert(kKeys * CH % 128 == 0, "whole chunks per thread");
    int* rows = reinterpret_cast<int*>(sm + L::ROWS);
    // Loads run ahead of the arithmetic: a tile's chunks wait in registers
    // while the tile before it is worked on, and the first warp looks its
    // keys' pool rows up one tile earlier still (-1: past the end).
    auto lookup = [&](int64_t key0) -> int {
      const int64_t key = key0 + tid;
      if (key >= k1) return -1;
      const int64_t page = key >> p.s_shift;
      int64_t phys = page < tlen ? load_index(table, page * tstride, ti64) : -1;
      if (phys < 0 || phys >= p.P) {
        report(p.status, B200_DEV_BAD_BLOCK);
        phys = 0;  // an in-bounds page; the status word tells
      }
      return static_cast<int>(p.layer_row0 + phys * p.S + (key & (p.S - 1)));
    };
    uint4 ck[IT], cv[IT];
    auto fetch = [&](const int* tile_rows) {
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int at = tid + 128 * i, r = at / CH, d0 = (at % CH) * E;
        const int row = tile_rows[r];
        ck[i] = cv[i] = make_uint4(0, 0, 0, 0);  // keys past the end, columns past D
        if (row >= 0 && d0 < p.D) {
          const int64_t off = (static_cast<int64_t>(row) * p.Hkv + g) * p.D + d0;
          ck[i] = __ldg(reinterpret_cast<const uint4*>(kp + off));
          cv[i] = __ldg(reinterpret_cast<const uint4*>(vp + off));
        }
      }
    };
    if (tid < kKeys) {
      rows[tid] = lookup(k0);
      rows[kKeys + tid] = lookup(k0 + kKeys);
    }
    __syncthreads();
    fetch(rows);

    int buf = 0;
    for (int64_t key0 = k0; key0 < k1; key0 += kKeys, buf ^= 1) {
      __syncthreads();  // the tile before is done with K and V
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int at = tid + 128 * i, r = at / CH, d0 = (at % CH) * E;
        float fk[E], fv[E];
        Elem<KV>::unpack(ck[i], fk);
        Elem<KV>::unpack(cv[i], fv);
#pragma unroll
        for (int e = 0; e < E; e += 4) {
          *reinterpret_cast<float4*>(K + r * L::LD + d0 + e) =
              make_float4(fk[e], fk[e + 1], fk[e + 2], fk[e + 3]);
          *reinterpret_cast<float4*>(V + r * L::LD + d0 + e) =
              make_float4(fv[e], fv[e + 1], fv[e + 2], fv[e + 3]);
        }
      }
      if (key0 + kKeys < k1) fetch(rows + (buf ^ 1) * kKeys);
      const int ahead = tid < kKeys ? lookup(key0 + 2 * kKeys) : -1;
      __syncthreads();
      // Scores: rows tr * RT + i, keys tc + TC * j.
      float2 s2[RT][KPT];
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < KPT; ++j) s2[i][j] = make_float2(0.f, 0.f);
#pragma unroll 4
      for (int d = 0; d < DP; d += 4) {
        float4 a[RT], b[KPT];
#pragma unroll
        for (int i = 0; i < RT; ++i)
          a[i] = *reinterpret_cast<const float4*>(Q + (tr * RT + i) * L::LD + d);
#pragma unroll
        for (int j = 0; j < KPT; ++j)
          b[j] = *reinterpret_cast<const float4*>(K + (tc + TC * j) * L::LD + d);
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
          for (int j = 0; j < KPT; ++j) {
            s2[i][j] = ffma2(make_float2(a[i].x, a[i].y), make_float2(b[j].x, b[j].y), s2[i][j]);
            s2[i][j] = ffma2(make_float2(a[i].z, a[i].w), make_float2(b[j].z, b[j].w), s2[i][j]);
          }
      }
      const int nkeys = static_cast<int>(min(k1 - key0, static_cast<int64_t>(kKeys)));
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        float s[KPT], mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < KPT; ++j) {
          s[j] = tc + TC * j < nkeys ? s2[i][j].x + s2[i][j].y : -INFINITY;
          mx = fmaxf(mx, s[j]);
        }
#pragma unroll
        for (int w = TC / 2; w >= 1; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
        const float mn = fmaxf(m[i], mx);
        const float ref = mn == -INFINITY ? 0.f : mn;  // all scores -inf: p = 0, not NaN
        const float alpha = exp2f(m[i] - ref);
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < KPT; ++j) {
          const float e = exp2f(s[j] - ref);
          sum += e;
          Pm[(tr * RT + i) * L::LP + tc + TC * j] = e;
        }
#pragma unroll
        for (int w = TC / 2; w >= 1; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
        l[i] = l[i] * alpha + sum;
        m[i] = mn;
#pragma unroll
        for (int c = 0; c < NG; ++c) {
          o[i][c].x *= alpha;
          o[i][c].y *= alpha;
          o[i][c].z *= alpha;
          o[i][c].w *= alpha;
        }
      }
      __syncwarp();  // a row's probabilities stay within its warp
#pragma unroll 4
      for (int j = 0; j < kKeys; ++j) {
        float4 v[NG];
#pragma unroll
        for (int c = 0; c < NG; ++c)
          if ((tc + TC * c) * 4 < DP)
            v[c] = *reinterpret_cast<const float4*>(V + j * L::LD + (tc + TC * c) * 4);
#pragma unroll
        for (int i = 0; i < RT; ++i) {
          const float pr = Pm[(tr * RT + i) * L::LP + j];
          const float2 p2 = make_float2(pr, pr);
#pragma unroll
          for (int c = 0; c < NG; ++c) {
            if ((tc + TC * c) * 4 >= DP) continue;
            const float2 lo = ffma2(p2, make_float2(v[c].x, v[c].y), make_float2(o[i][c].x, o[i][c].y));
            const float2 hi = ffma2(p2, make_float2(v[c].z, v[c].w), make_float2(o[i][c].z, o[i][c].w));
            o[i][c] = make_float4(lo.x, lo.y, hi.x, hi.y);
          }
        }
      }
      if (tid < kKeys) rows[buf * kKeys + tid] = ahead;
    }
  }

  // The rows' parts into slot `slot`.
  __device__ void write(const SharedParams& p, int g, int row0, int nrows, int slot) {
    const int tr = threadIdx.x / TC, tc = threadIdx.x % TC;
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const int r = tr * RT + i;
      if (r >= nrows) continue;
      const int64_t at = (static_cast<int64_t>(g) * p.rows + row0 + r) * p.ns + slot;
#pragma unroll
      for (int c = 0; c < NG; ++c) {
        const int d = (tc + TC * c) * 4;
        if (d < p.D) *reinterpret_cast<float4*>(p.acc + at * p.D + d) = o[i][c];
      }
      if (tc == 0) {
        p.ml[at * 2] = m[i];
        p.ml[at * 2 + 1] = l[i];
      }
    }
  }
};

// Prefix: CTA (part, row tile, key head).
template <typename KV, int R, int DP>
__global__ void __launch_bounds__(128) shared_prefix_elem_kernel(const __grid_constant__ SharedParams p,
                                                                const int counters) {
  let_next_start();
  extern __shared__ float4 sm4[];
  float* sm = reinterpret_cast<float*>(sm4);
  const int64_t cta = blockIdx.x + static_cast<int64_t>(gridDim.x) * (blockIdx.y + static_cast<int64_t>(gridDim.y) * blockIdx.z);
  for (int64_t i = cta * 128 + threadIdx.x; i < counters; i += static_cast<int64_t>(gridDim.x) * gridDim.y * gridDim.z * 128)
    p.cnt[i] = 0;  // of the own-key kernel
  const int part = blockIdx.x, row0 = blockIdx.y * R, g = blockIdx.z;
  const int64_t k0 = static_cast<int64_t>(part) * p.prefix_per;
  const int64_t k1 = min(p.prefix, k0 + p.prefix_per);
  const int nrows = min(R, p.rows - row0);
  ElemAttend<KV, R, DP> a;
  a.run(p, sm, g, row0, nrows, k0, k1, p.prefix_table, p.pt_stride, p.pt_i64,
        (p.prefix + p.S - 1) >> p.s_shift);
  a.write(p, g, row0, nrows, part);
}

// Own keys and the join: CTA ((sequence, key head, chunk of 8 rows), part).
template <typename KV, int DP>
__global__ void __launch_bounds__(128) shared_own_elem_kernel(const __grid_constant__ SharedParams p) {
  constexpr int R = kOwnRows;
  extern __shared__ float4 sm4[];
  float* sm = reinterpret_cast<float*>(sm4);
  __shared__ int last;
  int64_t idx = blockIdx.x;
  const int split = static_cast<int>(idx % p.own_splits);
  idx /= p.own_splits;
  const int64_t unit = idx;
  const int chunk = static_cast<int>(idx % p.row_chunks);
  idx /= p.row_chunks;
  const int g = static_cast<int>(idx % p.Hkv);
  const int b = static_cast<int>(idx / p.Hkv);
  const int row0 = b * p.rep + chunk * R;
  const int nrows = min(R, p.rep - chunk * R);
  const int64_t ctx = load_index(p.lens, b * p.len_stride, p.lens_i64);
  if (ctx < 1 || ctx < p.prefix || ctx > p.table_width * p.S) {
    if (split == 0) {
      if (threadIdx.x == 0) report(p.status, B200_DEV_BAD_LENGTH);
      if (p.out == p.q) wait_for_previous();  // it reads these rows
      for (int i = threadIdx.x; i < nrows * p.D; i += 128)
        store_elem(p.out, b * p.os0 + (g * p.rep + chunk * R + i / p.D) * p.os1 + (i % p.D) * p.os2,
                   p.out_dtype, 0.f);
    }
    end_after_previous();
    return;
  }
  int64_t k0, k1;
  const int parts = own_range(p, ctx - p.prefix, split, &k0, &k1);
  if (split >= parts) {
    end_after_previous();
    return;
  }
  ElemAttend<KV, R, DP> a;
  const int64_t row_bytes = p.tables_i64 ? 8 : 4;
  a.run(p, sm, g, row0, nrows, p.prefix + k0, p.prefix + k1,
        static_cast<const char*>(p.tables) + b * p.ts0 * row_bytes, p.ts1, p.tables_i64,
        p.table_width);
  a.write(p, g, row0, nrows, p.np + split);
  wait_for_previous();  // for the counters and the prefix's parts
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(&p.cnt[unit], 1) == parts - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  static_assert(ElemSmem<R, DP>::ROWS >= kJoinFloats, "the join's shared memory");
  join_rows(p, g, row0, nrows, parts, sm);
}

// ------------------------------------------------------------------ host
struct SharedPlan {
  bool mma;  // own keys by warp-level products,
  bool few;  // the prefix too
  bool tc;   // or on tcgen05
  TcSplit split;
  int np, own_splits, own_min, row_chunks;
  int64_t prefix_per;
  size_t acc_bytes, ml_bytes, cnt_bytes;
  size_t bytes() const { return acc_bytes + ml_bytes + cnt_bytes; }
};

size_t round256(size_t n) { return (n + 255) & ~size_t(255); }

// The parts of a call, from its sizes alone.
SharedPlan make_plan(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t prefix, int64_t max_own,
                     int64_t S, int kv_dtype, int q_dtype, int num_sms) {
  SharedPlan pl{};
  // A bf16 pool's products run on tensor cores: the large tiles take bf16
  // queries, the warp-level form any, f16 and f32 ones in exact pieces.  f32
  // pools would lose bits there.
  // (Pages of fewer than 8 tokens would make swizzled boxes of less than 1 KB.)
  pl.mma = kv_dtype == B200_DTYPE_BF16 && S >= 8;
  const int64_t rep = Hq / Hkv, rows = B * rep;
  const bool mma = pl.mma;
  // Few rows leave most of a tensor tile empty: there the prefix is worked off
  // eight rows at a time like own keys, which reads it (from L2) once for each
  // eight.  That starts and ends faster and is up to 16 rows ahead at any length
  // (4 sequences of 8 x 4 heads over 2048 keys: 10 us against 15; over 32768: 32
  // against 43; 1 of 32 x 1: 83 against 116).  Above, it is as long as little is
  // read: 64 rows to each of 8 heads, 1024 keys 13 us against 17, 2048 the same,
  // 8192 30 against 23.  Queries of other types have no tensor-tile form, however
  // many: eight rows at a time they take 245 (f16) and 280 us (f32) at 1024 rows to
  // each of 8 heads behind 4096 keys, by f32 arithmetic 694.
  const int64_t eights = ceil_div(rows, kOwnRows) * Hkv;
  pl.few = mma && prefix > 0 &&
           (q_dtype != B200_DTYPE_BF16 || rows <= 16 || eights * prefix < (int64_t(1) << 17));
  pl.tc = mma && prefix > 0 && !pl.few;
  // Prefix: parts of whole key tiles that give about two CTAs per SM.
  pl.np = 0;
  pl.prefix_per = 0;
  if (pl.tc) {
    pl.split = shared_tc_split(rows, Hkv, prefix, num_sms);
    pl.np = pl.split.np;
  } else if (pl.few) {
    // Two CTAs per SM, three where much is read more than once; at least 64
    // keys a part, above 16 parts, which the join has to read, 256 (2048 keys of
    // 8 heads: 16 parts 9.8 us, 8 and 32 parts 10.8), and above 32 parts 1024
    // (131072 keys of 2 heads: 64 parts 43 us, 32 parts 59; 32768 keys of 4: 29
    // and 26).
    const int per_sm = rows <= 8 || eights * prefix < (int64_t(1) << 18) ? 2 : 3;
    int64_t parts = std::min({per_sm * num_sms / eights, ceil_div(prefix, 64),
                              std::max({int64_t(16), std::min<int64_t>(ceil_div(prefix, 256), 32),
                                        std::min<int64_t>(ceil_div(prefix, 1024), kPrefixParts)})});
    parts = std::max(parts, std::min<int64_t>(ceil_div(prefix, 4096), 32));
    pl.prefix_per = ceil_div(ceil_div(prefix, parts), 16) * 16;
    pl.np = static_cast<int>(ceil_div(prefix, pl.prefix_per));
  } else if (prefix > 0) {
    const int64_t units = ceil_div(rows, 64) * Hkv;
    int64_t parts = std::min<int64_t>(ceil_div(2 * num_sms, units), ceil_div(prefix, 4 * kKeys));
    parts = std::max<int64_t>(1, std::min<int64_t>(parts, kPrefixParts));
    pl.prefix_per = ceil_div(ceil_div(prefix, parts), kKeys) * kKeys;
    pl.np = static_cast<int>(ceil_div(prefix, pl.prefix_per));
  }
  // Own keys: enough parts to fill the GPU, of about 1024 keys at most while
  // there are no more than kOwnParts of them (131072 own keys: 4096 each).  The
  // lengths are the device's, and a part that a sequence does not need is a CTA
  // that reads its length and ends, so that tables much wider than the lengths cost
  // time: at most 28 rounds of the four CTAs to an SM.  (256 sequences of 8 heads
  // with up to 128 own keys and tables for 131072: 83 us, with 32 parts 154, tables
  // for no more than the lengths 61; one of them with 16384 own keys, tables for
  // 32768: 89 and 149; one with 100000: 309 and 195.)
  pl.row_chunks = static_cast<int>(ceil_div(rep, kOwnRows));
  pl.own_min = mma ? 128 : 64;
  const int64_t units = B * Hkv * pl.row_chunks;
  int64_t splits = std::max<int64_t>(ceil_div(2 * num_sms, units), ceil_div(max_own, 1024));
  splits = std::min<int64_t>({splits, ceil_div(max_own, pl.own_min), int64_t(kOwnParts),
                              std::max<int64_t>(28 * 4 * num_sms / units, 1)});
  pl.own_splits = static_cast<int>(std::max<int64_t>(splits, 1));
  const size_t slots = static_cast<size_t>(Hkv * rows) * (pl.np + pl.own_splits);
  pl.acc_bytes = round256(slots * D * sizeof(float));
  pl.ml_bytes = round256(slots * 2 * sizeof(float));
  pl.cnt_bytes = round256(static_cast<size_t>(units) * sizeof(int32_t));
  return pl;
}

// Raises the kernel's shared memory limit once per device (`state` is the
// kernel's own).
template <typename Kernel>
int allow_smem(Kernel kern, int bytes, int device, std::atomic<int>* state) {
  if (bytes <= 48 * 1024 || (device < 64 && state[device].load(std::memory_order_acquire))) return B200_OK;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(shared prefix)");
  if (device < 64) state[device].store(1, std::memory_order_release);
  return B200_OK;
}

template <typename KV, int R, int DP>
int launch_prefix_rows(const SharedParams& p, const SharedPlan& pl, int counters, int device,
                       cudaStream_t stream) {
  const int64_t tiles = ceil_div(p.rows, R);
  if (tiles > 65535) return fail(B200_ERR_UNSUPPORTED, "shared prefix: too many query rows");
  auto kern = shared_prefix_elem_kernel<KV, R, DP>;
  static std::atomic<int> state[64];
  int rc = allow_smem(kern, ElemSmem<R, DP>::BYTES, device, state);
  if (rc != B200_OK) return rc;
  const dim3 grid(static_cast<unsigned>(pl.np), static_cast<unsigned>(tiles),
                  static_cast<unsigned>(p.Hkv));
  kern<<<grid, 128, ElemSmem<R, DP>::BYTES, stream>>>(p, counters);
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? B200_OK : cuda_fail(e, "shared prefix launch");
}

template <typename KV, int DP>
int launch_prefix_elem(const SharedParams& p, const SharedPlan& pl, int counters, int device,
                       cudaStream_t stream) {
  // Few rows would leave most of a tile of 64 empty (16 sequences of 8 heads
  // of 32 over 4093 fp32 keys: 13 us, with 64 rows 17 us).
  if (p.rows <= 16) return launch_prefix_rows<KV, 16, DP>(p, pl, counters, device, stream);
  return launch_prefix_rows<KV, 64, DP>(p, pl, counters, device, stream);
}

template <typename KV, int DP>
int launch_own_elem(const SharedParams& p, bool overlap, int device, cudaStream_t stream) {
  const int64_t grid = static_cast<int64_t>(p.B) * p.Hkv * p.row_chunks * p.own_splits;
  if (grid > 0x7fffffffLL) return fail(B200_ERR_UNSUPPORTED, "shared prefix: grid too large");
  auto kern = shared_own_elem_kernel<KV, DP>;
  static std::atomic<int> state[64];
  int rc = allow_smem(kern, ElemSmem<8, DP>::BYTES, device, state);
  if (rc != B200_OK) return rc;
  return launch_own(kern, grid, 128, ElemSmem<8, DP>::BYTES, stream, overlap, p);
}

template <typename KV>
int launch_prefix_elem_d(const SharedParams& p, const SharedPlan& pl, int counters, int device,
                         cudaStream_t stream) {
  if (p.D <= 32) return launch_prefix_elem<KV, 32>(p, pl, counters, device, stream);
  if (p.D <= 64) return launch_prefix_elem<KV, 64>(p, pl, counters, device, stream);
  return launch_prefix_elem<KV, 128>(p, pl, counters, device, stream);
}

template <typename KV>
int launch_own_elem_d(const SharedParams& p, bool overlap, int device, cudaStream_t stream) {
  if (p.D <= 32) return launch_own_elem<KV, 32>(p, overlap, device, stream);
  if (p.D <= 64) return launch_own_elem<KV, 64>(p, overlap, device, stream);
  return launch_own_elem<KV, 128>(p, overlap, device, stream);
}

}  // namespace

size_t shared_prefix_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t prefix,
                                     int64_t table_width, int64_t S, int kv_dtype, int q_dtype,
                                     int num_sms) {
  const int64_t own = std::max<int64_t>(table_width * S - prefix, 0);
  return make_plan(B, Hq, Hkv, D, prefix, own, S, kv_dtype, q_dtype, num_sms).bytes();
}

int launch_shared_prefix(const b200_shared_prefix_args_t& a, cudaStream_t stream) {
  DeviceInfo dev;
  int rc = current_device_info(&dev);
  if (rc != B200_OK) return rc;
  const int64_t B = a.batch, Hq = a.num_q_heads, Hkv = a.pool.num_heads, D = a.pool.head_dim;
  const int64_t S = a.pool.block_size;
  const int64_t own = std::max<int64_t>(a.table_width * S - a.prefix_len, 0);
  const SharedPlan pl = make_plan(B, Hq, Hkv, D, a.prefix_len, own, S, a.pool.dtype, a.q_dtype,
                                  dev.num_sms);
  if (a.workspace == nullptr || a.workspace_bytes < pl.bytes()) {
    char buf[160];
    snprintf(buf, sizeof(buf), "shared prefix decode needs %zu workspace bytes, got %zu", pl.bytes(),
             a.workspace_bytes);
    return fail(B200_ERR_WORKSPACE, buf);
  }
  if (pl.np > kPrefixParts || pl.own_splits > kOwnParts)
    return fail(B200_ERR_UNSUPPORTED, "shared prefix: too many parts");
  SharedParams p{};
  p.q = a.q;
  p.out = a.out;
  p.qs0 = a.q_stride[0], p.qs1 = a.q_stride[1], p.qs2 = a.q_stride[2];
  p.os0 = a.out_stride[0], p.os1 = a.out_stride[1], p.os2 = a.out_stride[2];
  p.k_pool = a.pool.k;
  p.v_pool = a.pool.v;
  p.P = a.pool.num_blocks;
  p.S = S;
  p.layer_row0 = a.layer_idx * p.P * S;
  p.prefix_table = a.prefix_table;
  p.pt_stride = a.prefix_table_stride;
  p.pt_i64 = a.prefix_table_dtype == B200_INDEX_I64;
  p.tables = a.block_tables;
  p.ts0 = a.block_table_stride[0];
  p.ts1 = a.block_table_stride[1];
  p.tables_i64 = a.block_table_dtype == B200_INDEX_I64;
  p.table_width = a.table_width;
  p.lens = a.context_lengths;
  p.len_stride = a.context_length_stride;
  p.lens_i64 = a.context_length_dtype == B200_INDEX_I64;
  uint8_t* ws = static_cast<uint8_t*>(a.workspace);
  p.acc = reinterpret_cast<float*>(ws);
  p.ml = reinterpret_cast<float*>(ws + pl.acc_bytes);
  p.cnt = reinterpret_cast<int32_t*>(ws + pl.acc_bytes + pl.ml_bytes);
  p.status = a.status;
  p.prefix = a.prefix_len;
  p.B = static_cast<int32_t>(B);
  p.Hq = static_cast<int32_t>(Hq);
  p.Hkv = static_cast<int32_t>(Hkv);
  p.D = static_cast<int32_t>(D);
  p.rep = static_cast<int32_t>(Hq / Hkv);
  p.rows = p.B * p.rep;
  p.s_shift = log2i(S);
  p.np = pl.np;
  p.ns = pl.np + pl.own_splits;
  p.prefix_per = static_cast<int32_t>(pl.prefix_per);
  p.own_splits = pl.own_splits;
  p.own_min = pl.own_min;
  p.row_chunks = pl.row_chunks;
  p.q_dtype = a.q_dtype;
  p.out_dtype = a.out_dtype;
  p.qscale = static_cast<float>(1.4426950408889634 / sqrt(static_cast<double>(D)));
  // The parts of a sequence's own keys count themselves; the prefix's kernel,
  // where there is one, clears the counters on its way.
  const int counters = pl.mma && pl.own_splits == 1 ? 0 : static_cast<int>(pl.cnt_bytes / sizeof(int32_t));
  if (counters > 0 && pl.np == 0) {
    cudaError_t e = cudaMemsetAsync(p.cnt, 0, pl.cnt_bytes, stream);
    if (e != cudaSuccess) return cuda_fail(e, "cudaMemsetAsync(shared prefix counters)");
  }
  const bool f32 = a.pool.dtype == B200_DTYPE_F32;
  if (pl.tc)
    rc = launch_shared_prefix_tc(p, a.pool, pl.split, counters, stream);
  else if (pl.few)
    rc = launch_shared_prefix_mma(p, a.pool, counters, stream);
  else if (pl.np > 0)
    rc = f32 ? launch_prefix_elem_d<float>(p, pl, counters, dev.device, stream)
             : launch_prefix_elem_d<__nv_bfloat16>(p, pl, counters, dev.device, stream);
  if (rc != B200_OK) return rc;
  const bool overlap = pl.np > 0;
  if (pl.mma) return launch_shared_own_mma(p, a.pool, overlap, stream);
  return f32 ? launch_own_elem_d<float>(p, overlap, dev.device, stream)
             : launch_own_elem_d<__nv_bfloat16>(p, overlap, dev.device, stream);
}

}  // namespace b200
