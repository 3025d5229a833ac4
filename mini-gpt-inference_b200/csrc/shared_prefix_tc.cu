// shared_prefix_tc.cu -- the prefix's part of the shared-prefix decode on
// tcgen05 tensor cores (bf16 pools and queries, block size >= 8, and rows and
// keys enough).
//
// For a key head g the rows q[b, h] of all sequences and of g's query heads
// form one matrix of B * rep rows: S = Q K^T, P = 2^(S - max), O = P V over
// the prefix.  A unit is up to 256 of these rows (two tiles of 128) of one key
// head; its key tiles of 128 are read once for both.  The units' key tiles,
// end to end, are cut into equal runs, one per CTA and SM, so that every CTA
// has the same work whatever the batch, heads and prefix are; a run that
// crosses units is worked off in segments, each of which leaves its rows'
// unnormalised O, maximum and sum in a slot of the workspace.
//
// Roles (12 warps):
//   warp 0      loads K and V tiles by TMA, page by page, into one ring
//               (K of a tile, then its V);
//   warp 1      issues every product.  The tensor pipe runs the products of
//               one thread in order, so S of the next tile may follow P V of
//               this one into the same TMEM columns without a wait, and the
//               barrier that announces S(k + 1) also says that P V(k) is done;
//   warps 4-7, 8-11  softmax of row tile 0 / 1: thread r owns row r = TMEM
//               lane r; reads its scores, writes its weights as bf16 over them.
// While one tile's softmax runs, the tensor pipe works on the other's S and
// P V.  With at most 128 rows there is one row tile and the two softmax groups
// take its key tiles in turn, each with its own O; group 0 adds them up.
//
// The weights are rounded to bf16 for P V.  Two row tiles are bound by the
// products and leave it at that (error of bf16 outputs against 64 bits 0.0023);
// one row tile is bound by the bytes, and what the rounding left takes part as a
// second bf16 product (0.0017: rows differ from exact ones by their own rounding
// alone).  In two row tiles the second product costs 12 to 18 %: 64 sequences over
// 32768 keys 67 to 79 us, 256 over 16384 129 to 149.
//
// TMEM (512 columns): S_w / P_w at 128 w, O_w at 256 + 128 w.
// V rows behind the prefix are cleared in shared memory before they are
// used: unwritten pool rows can hold NaN, and 0 * NaN is NaN.
// Every wait is bounded and a whole warp's decision; after one runs out all
// roles leave.
//
// Measured (32 query heads of 128 over 8 key heads): 256 sequences over 16384
// keys 73 us, of which 53 us are 28 tile pairs of 1.9 us a CTA (the products
// alone, at this GPU's rate for them, 1.4 us) and the rest the segments'
// beginnings and ends; 64 over 32768 45 us (21 us at the copy rate).  A softmax
// of two threads to a row (16 warps), of rows whose weights go to the products
// quarter by quarter, of weights by polynomial on the FMA pipes, and turns of
// the two groups at the exponential unit were all built and measured: 2 to 2.6
// us a tile pair.
#include <float.h>
#include <math.h>

#include <algorithm>
#include <atomic>

#include "common.cuh"
#include "host_util.h"
#include "kernels.h"
#include "shared_prefix.cuh"
#include "tcgen05.cuh"

namespace b200 {
namespace {

constexpr int kBM = 128, kBN = 128;
constexpr int kThreads = 384;

struct TcParams {
  SharedParams s;
  int64_t units;
  int32_t unit_tiles;  // key tiles per unit
  int32_t unit_pairs;  // units per key head
  int32_t rbox, rb_shift;
  int32_t q_vec;
  int32_t zero_count;  // counters to clear for the own-key kernel
};

template <int DP>
struct TcSmem {
  static constexpr int HALVES = DP / 64;
  static constexpr int HALF = 128 * 128;       // 128 rows of 128 bytes
  static constexpr int TILE = HALVES * HALF;   // a row or key tile
  static constexpr int STAGES = DP == 128 ? 5 : 10;
  static constexpr int Q0 = 0;
  static constexpr int RING = 2 * TILE;
  static constexpr int BAR = RING + STAGES * TILE;
  static constexpr int BYTES = BAR + 512;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A whole warp's bounded wait: all lanes get one answer.  What a warp does next
// (votes, elections, TMEM access) needs every lane, and lanes that poll for
// themselves may pass the limit, or see another role's abort flag, on different
// sides of it.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity)) != 0;
}
// The same; no also where a role has given up.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, const volatile int32_t* abort_flag) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity) && *abort_flag == 0) != 0;
}

// Weights 2^(v scale - ref) of 32 scores as bf16 pairs; returns their sum
// before the rounding.  LO: rounded towards zero, and also what that left.
template <bool LO>
__device__ __forceinline__ float weights32(const float* v, float scale, float ref, uint32_t* pk, uint32_t* lo) {
  const float2 sc2 = make_float2(scale, scale), nm2 = make_float2(-ref, -ref), one2 = make_float2(1.f, 1.f);
  const float2 minus2 = make_float2(-1.f, -1.f), keep2 = make_float2(kKeepSign, kKeepSign);
  float2 q[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) q[e] = ffma2(make_float2(v[2 * e], v[2 * e + 1]), sc2, nm2);
#pragma unroll
  for (int e = 0; e < 16; ++e) q[e] = make_float2(ex2(q[e].x), ex2(q[e].y));
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    if constexpr (LO) {
      pk[e] = chop_bf16(q[e].x, q[e].y);
      const float2 rest = ffma2(q[e], keep2, ffma2(bf16x2_to_float2(pk[e]), minus2, q[e]));
      lo[e] = pack_bf16(rest.x, rest.y);
    } else {
      pk[e] = pack_bf16(q[e].x, q[e].y);
    }
  }
#pragma unroll
  for (int w = 8; w >= 1; w >>= 1)
#pragma unroll
    for (int e = 0; e < w; ++e) q[e] = ffma2(q[e], one2, q[e + w]);
  return q[0].x + q[0].y;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Byte offset of 16-byte chunk ch of row r in a 128-byte-swizzled half tile.
__device__ __forceinline__ uint32_t sw128(int r, int ch) {
  return static_cast<uint32_t>(r) * 128u + (static_cast<uint32_t>(ch ^ (r & 7)) << 4);
}

// What a segment costs besides its tiles (queries in, rows out, the first
// scores), in tiles: 11 us against 1.9 us a tile.  (64 sequences over 32k: 47.9
// us at 4, 45.5 us at 6; 256 over 16k the same.)
constexpr int kSegment = 6;

// Runs of equal cost: a unit's tiles, then the segment's cost, is a stretch of
// unit_tiles + kSegment; the stretches, end to end, are cut evenly.
__host__ __device__ inline int64_t run_begin(int64_t units, int unit_tiles, int64_t cta, int64_t ctas) {
  const int64_t stretch = unit_tiles + kSegment;
  const int64_t x = units * stretch * cta / ctas;
  const int64_t unit = x / stretch, off = x - unit * stretch;
  return unit * unit_tiles + (off < unit_tiles ? off : unit_tiles);
}
// The CTA that has tile `tile` of unit `unit`: the last that begins at or before it.
__host__ __device__ inline int64_t cta_of(int64_t units, int unit_tiles, int64_t ctas, int64_t unit, int tile) {
  const int64_t stretch = unit_tiles + kSegment;
  return ((unit * stretch + tile + 1) * ctas - 1) / (units * stretch);
}

// A CTA's run of key tiles, segment by segment.
struct Segments {
  int64_t pos, end;
  int tiles_per_unit;
  int unit, j0, n;  // this segment: key tiles [j0, j0 + n) of a unit
  __device__ Segments(const TcParams& p) {
    pos = run_begin(p.units, p.unit_tiles, blockIdx.x, gridDim.x);
    end = run_begin(p.units, p.unit_tiles, blockIdx.x + 1, gridDim.x);
    tiles_per_unit = p.unit_tiles;
  }
  __device__ bool next() {
    if (pos >= end) return false;
    unit = static_cast<int>(pos / tiles_per_unit);
    j0 = static_cast<int>(pos - static_cast<int64_t>(unit) * tiles_per_unit);
    n = static_cast<int>(min(static_cast<int64_t>(tiles_per_unit - j0), end - pos));
    pos += n;
    return true;
  }
};

// The 32 query rows from row0 on of key head g (zeros from `rows` on) into
// rows r0 .. r0 + 31 of a swizzled tile, by one warp: whole rows by neighbouring
// lanes, all loads on their way before the first store.  (A row per lane, 32
// lines to a load, took 7 us for both tiles; this takes 3.)
template <int DP>
__device__ __forceinline__ void load_q_rows(uint8_t* tile, int r0, const SharedParams& s, int row0, int g,
                                            int q_vec) {
  constexpr int CH = DP / 8;       // chunks per row
  constexpr int RPI = 32 / CH;     // rows per load
  constexpr int IT = 32 / RPI;
  const int lane = threadIdx.x & 31;
  const int mine = min(row0 + lane, s.rows - 1);
  const int b = mine / s.rep;
  const int64_t off = b * s.qs0 + static_cast<int64_t>(g * s.rep + mine - b * s.rep) * s.qs1;
  const int c = lane % CH;
  const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(s.q);
  uint4 w[IT];
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int r = i * RPI + lane / CH;
    const __nv_bfloat16* src = q + __shfl_sync(0xffffffffu, off, r);
    w[i] = make_uint4(0, 0, 0, 0);
    if (row0 + r < s.rows && c * 8 < s.D) {
      if (q_vec) {
        w[i] = *reinterpret_cast<const uint4*>(src + c * 8);
      } else {
        uint32_t x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const __nv_bfloat162 h =
              __halves2bfloat162(src[(c * 8 + 2 * e) * s.qs2], src[(c * 8 + 2 * e + 1) * s.qs2]);
          x[e] = *reinterpret_cast<const uint32_t*>(&h);
        }
        w[i] = make_uint4(x[0], x[1], x[2], x[3]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < IT; ++i)
    *reinterpret_cast<uint4*>(tile + (c >> 3) * (128 * 128) + sw128(r0 + i * RPI + lane / CH, c & 7)) = w[i];
}

// W columns (32 or 64) of a warp's 32 rows, a row per lane, to global rows of
// `pitch` floats through shared memory (32 x W floats, 16-byte chunks permuted
// by row so that neither side meets a bank twice): W / 4 neighbouring lanes
// write consecutive bytes of a row.  (16 bytes a lane, straight from the
// lane's row, took 9 us for both tiles; this takes 4.)
template <int W>
struct RowWriter {
  static constexpr int CH = W / 4;
  float* stage;
  float* dst;  // row 0, column 0
  int64_t pitch;
  int rows, cols;  // that exist
  __device__ __forceinline__ void put(int c0, const float* o) {  // columns c0 .. c0 + 31 of this row
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int e = 0; e < 32; e += 4) {
      const int ch = (c0 % W + e) >> 2;
      *reinterpret_cast<float4*>(stage + lane * W + ((ch ^ (lane & (CH - 1))) << 2)) =
          make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
    }
  }
  __device__ __forceinline__ void flush(int c0) {  // columns c0 .. c0 + W - 1
    const int lane = threadIdx.x & 31;
    const int ch = lane % CH;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int r = i * (32 / CH) + lane / CH;
      const float4 v = *reinterpret_cast<const float4*>(stage + r * W + ((ch ^ (r & (CH - 1))) << 2));
      if (r < rows && c0 + ch * 4 < cols)
        *reinterpret_cast<float4*>(dst + r * pitch + c0 + ch * 4) = v;
    }
    __syncwarp();
  }
};

// ONE: at most 128 rows per key head.
template <int DP, bool ONE>
__global__ void __launch_bounds__(kThreads, 1)
    shared_prefix_tc_kernel(const __grid_constant__ CUtensorMap tmk,
                            const __grid_constant__ CUtensorMap tmv, const __grid_constant__ TcParams p) {
  using L = TcSmem<DP>;
  constexpr int NS = L::STAGES;
  const SharedParams& s = p.s;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::BAR);  // [NS]
  uint64_t* empty = full + NS;                                  // [NS]
  uint64_t* q_full = empty + NS;                                // [2]
  uint64_t* s_full = q_full + 2;                                // [2]
  uint64_t* p_full = s_full + 2;                                // [2]
  uint64_t* o_full = p_full + 2;                                // [2]
  uint64_t* merge_full = o_full + 2;
  uint64_t* merge_done = merge_full + 1;
  uint64_t* drained = merge_done + 1;                           // [2]
  uint64_t* idle = drained + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(idle + 1);
  volatile int32_t* abort_flag = reinterpret_cast<int32_t*>(idle + 2);
  static_assert((2 * NS + 15) * 8 <= 512, "barrier area too small");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  let_next_start();
  if (threadIdx.x == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int w = 0; w < 2; ++w) {
      mbar_init(&q_full[w], 128);
      mbar_init(&s_full[w], 1);
      mbar_init(&p_full[w], 4);  // a lane of each warp
      mbar_init(&o_full[w], 1);
      mbar_init(&drained[w], 128);
    }
    mbar_init(merge_full, 256);
    mbar_init(merge_done, 256);
    mbar_init(idle, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_slot)),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  constexpr bool one = ONE;
  auto unit_rows = [&](int unit) { return (unit % p.unit_pairs) * 2 * kBM; };  // its first row
  auto give_up = [&]() {
    report(s.status, B200_DEV_WAIT_TIMEOUT);
    *abort_flag = 1;
  };

  // Registers: 384 threads start with 168 each (64512 in all); 128 x 56 +
  // 256 x 224 is the same sum.  A softmax thread works on a row of 128 scores.
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 0) {
      // ------------------------------------------------------------ loads
      const int box_bytes = 64 * p.rbox * 2;
      const int boxes_per_tile = kBN / p.rbox;  // <= 16
      const int64_t table_len = (s.prefix + s.S - 1) >> s.s_shift;
      uint32_t it = 0;
      bool ok = true;
      Segments sg(p);
      while (ok && sg.next()) {
        const int g = sg.unit / p.unit_pairs;
        // Lane i looks up block i of a tile (16 at most), one tile ahead.
        auto blocks = [&](int j) {
          return static_cast<int>(min(static_cast<int64_t>(boxes_per_tile),
                                      (s.prefix - static_cast<int64_t>(j) * kBN + p.rbox - 1) >> p.rb_shift));
        };
        auto entry = [&](int j) -> int64_t {
          if (j >= sg.j0 + sg.n || lane >= blocks(j)) return 0;
          const int64_t page = (static_cast<int64_t>(j) * kBN + (static_cast<int64_t>(lane) << p.rb_shift)) >> s.s_shift;
          return page < table_len ? load_index(s.prefix_table, page * s.pt_stride, s.pt_i64) : -1;
        };
        int64_t next = entry(sg.j0);
        for (int j = sg.j0; ok && j < sg.j0 + sg.n; ++j) {
          const int nb = blocks(j);
          int64_t phys = next;
          next = entry(j + 1);
          if (lane < nb && (phys < 0 || phys >= s.P)) {
            report(s.status, B200_DEV_BAD_BLOCK);
            phys = 0;  // an in-bounds page; the status word tells
          }
          const int64_t key = static_cast<int64_t>(j) * kBN + (static_cast<int64_t>(lane) << p.rb_shift);
          const int row = static_cast<int>(s.layer_row0 + phys * s.S + (key & (s.S - 1)));
#pragma unroll
          for (int kv = 0; kv < 2; ++kv, ++it) {
            const int st = static_cast<int>(it % NS);
            ok = warp_wait(&empty[st], ((it / NS) & 1u) ^ 1u, abort_flag);
            if (!ok) break;
            if (lane == 0)
              mbar_arrive_expect_tx(&full[st], static_cast<uint32_t>(nb * L::HALVES * box_bytes));
            __syncwarp();
            if (lane < nb) {
              uint8_t* dst = smem + L::RING + st * L::TILE + lane * p.rbox * 128;
#pragma unroll
              for (int h = 0; h < L::HALVES; ++h)
                tma_load_3d(dst + h * L::HALF, kv == 0 ? &tmk : &tmv, &full[st], h * 64, g, row);
            }
          }
        }
      }
      // Copies in flight land before the CTA ends.
      for (uint32_t i = it > NS ? it - NS : 0; i < it; ++i) ok = warp_wait(&full[i % NS], (i / NS) & 1u) && ok;
      if (!ok && lane == 0) give_up();
    } else if (warp == 1) {
      // ------------------------------------------------------------ products
      // The whole warp, so that descriptors stay in uniform registers (one lane
      // issues), in small loops: this code shares its instruction cache with the
      // softmax warps, and a step that has to be fetched again is late.
      {
        constexpr uint32_t idesc_s = idesc_bf16(128, kBN, false);
        constexpr uint32_t idesc_o = idesc_bf16(128, DP, true);
        const uint64_t dq0 = smem_desc_sw128(smem_u32(smem + L::Q0), 16, 1024);
        const uint64_t dk0 = smem_desc_sw128(smem_u32(smem + L::RING), 16, 1024);
        const uint64_t dv0 = smem_desc_sw128(smem_u32(smem + L::RING), L::HALF, 1024);
        uint32_t first = 0;         // ring entry of the segment's first K
        uint32_t np0 = 0, np1 = 0;  // P tiles of group w awaited so far
        uint32_t nq0 = 0, nq1 = 0;  // Q tiles awaited so far
        bool ok = true;
        auto wait = [&](uint64_t* bar, uint32_t parity) { return warp_wait(bar, parity, abort_flag); };
        auto wait_entry = [&](uint32_t e) { return wait(&full[e % NS], (e / NS) & 1u); };
        Segments sg(p);
        while (ok && sg.next()) {
          const int n = sg.n;
          const bool two = !one && unit_rows(sg.unit) + kBM < s.rows;  // row tile 1 is there
          ok = wait(&q_full[0], nq0++ & 1u) && (!two || wait(&q_full[1], nq1++ & 1u));
          // Step t: P V of tile t, then S of tile t + lead for the same group, which
          // frees the columns in that order.  Two row tiles: both groups, one tile
          // ahead; one row tile: the groups alternate, two tiles ahead.
          const int lead = one ? 2 : 1, groups = two ? 2 : 1;
#pragma unroll 1
          for (int t = -lead; ok && t < n; ++t) {
            const uint32_t ev = first + 2 * t + 1, ek = first + 2 * (t + lead);
#pragma unroll 1
            for (int i = 0; ok && i < groups; ++i) {
              const int w = one ? t & 1 : i;
              const bool last = i == groups - 1;
              if (t >= 0) {
                ok = wait(&p_full[w], (w ? np1 : np0) & 1u) && (i > 0 || wait_entry(ev));
                if (!ok) break;
                (w ? np1 : np0) += 1;
                tc_fence_after();
                uint32_t tp = tmem + w * 128;
#pragma unroll 1
                for (int part = 0; part < (one ? 2 : 1); ++part) {
                  uint64_t dv = dv0 + static_cast<uint64_t>((ev % NS) * (L::TILE >> 4));
#pragma unroll 8
                  for (int kk = 0; kk < kBN / 16; ++kk, dv += 128, tp += 8)
                    mma_bf16_ts(tmem + 256 + w * 128, tp, dv, idesc_o, t >= lead || part + kk > 0 ? 1u : 0u);
                }
                if (last) mma_commit(&empty[ev % NS]);
                if (t + lead >= n) mma_commit(&o_full[w]);
              }
              if (t + lead < n) {
                ok = i > 0 || wait_entry(ek);
                if (!ok) break;
                tc_fence_after();
                uint64_t dq = dq0 + static_cast<uint64_t>(i * (L::TILE >> 4));
                uint64_t dk = dk0 + static_cast<uint64_t>((ek % NS) * (L::TILE >> 4));
#pragma unroll 8
                for (int kk = 0; kk < DP / 16; ++kk) {
                  mma_bf16(tmem + w * 128, dq, dk, idesc_s, kk > 0 ? 1u : 0u);
                  const uint64_t step = kk == 3 ? (L::HALF - 96) >> 4 : 2;  // 16 d on, or the other half
                  dq += step;
                  dk += step;
                }
                mma_commit(&s_full[w]);
                if (last) mma_commit(&empty[ek % NS]);
              }
            }
          }
          first += 2 * n;
        }
        if (!ok && lane == 0) give_up();
        mma_commit(idle);  // every product issued has ended before TMEM is freed
        if (!warp_wait(idle, 0) && lane == 0) report(s.status, B200_DEV_WAIT_TIMEOUT);
        __syncwarp();
      }
    } else {
      // Counters of the kernel that follows on the stream.
      for (int i = blockIdx.x * 64 + threadIdx.x - 64; i < p.zero_count; i += gridDim.x * 64) s.cnt[i] = 0;
    }
  } else {
    // ------------------------------------------------------------ softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    const int w = (warp - 4) >> 2;
    const int r = (warp & 3) * 32 + lane;  // row of the tile = TMEM lane
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + w * 128 + lanes, to = tmem + 256 + w * 128 + lanes;
    const float scale = s.qscale;
    uint32_t tiles = 0, oseg = 0, mseg = 0, dseg = 0;
    uint32_t first = 0;
    bool ok = true;
    Segments sg(p);
    while (ok && sg.next()) {
      const int n = sg.n;
      const int g = sg.unit / p.unit_pairs;
      const int tile_row0 = unit_rows(sg.unit) + (one ? 0 : w * kBM);
      const int row = tile_row0 + r;
      const bool group_live = tile_row0 < s.rows;  // uniform over the group
      const bool warp_live = tile_row0 + (warp & 3) * 32 < s.rows;
      const int cnt = one ? (n + 1 - w) / 2 : group_live ? n : 0;
      // Q: the last segment's S products have all ended (s_full, o_full, and
      // in the one-tile form merge_done), and so has the use of its memory below.
      if (one ? w == 0 : group_live) {
        load_q_rows<DP>(smem + L::Q0 + w * L::TILE, (warp & 3) * 32, s, tile_row0 + (warp & 3) * 32, g,
                        p.q_vec);
        fence_proxy_async_shared();
        mbar_arrive(&q_full[w]);
      }
      float m = -INFINITY, l = 0.f;
      for (int k = 0; k < cnt; ++k, ++tiles) {
        const int jj = one ? 2 * k + w : k;  // tile within the segment
        ok = warp_wait(&s_full[w], tiles & 1u, abort_flag);
        if (!ok) break;
        tc_fence_after();
        const int left = static_cast<int>(  // keys from here on
            min(s.prefix - static_cast<int64_t>(sg.j0 + jj) * kBN, static_cast<int64_t>(kBN)));
        if (warp_live) {
          // The weights are taken relative to the row's reference m as it stands,
          // and their sum tells whether that was far too low, or none yet (or a
          // score is not a number); the rare warp with such a row finds a new one and does
          // the tile again.  The first tile has no reference yet.  What runs
          // once or rarely is rolled up: cold instructions cost more than
          // loops here (unrolled, the first two tiles of a CTA took 11 us).
          if (left < kBN) {  // the prefix ends in this tile
#pragma unroll 1
            for (int c = 0; c < kBN; c += 32) {
              float v[32];
              tmem_ld32(ts + c, v);
              wait_ld32(v);
#pragma unroll
              for (int e = 0; e < 32; ++e) v[e] = c + e < left ? v[e] : -INFINITY;
              tmem_st32(ts + c, v);
            }
            tmem_wait_st();
          }
          uint32_t pk[kBN / 2], lo[ONE ? kBN / 2 : 1];
          float add, alpha = 1.f;
#pragma unroll 1
          for (bool fresh = k == 0;; fresh = true) {
            if (fresh) {
              float mx = -INFINITY;
#pragma unroll 1
              for (int c = 0; c < kBN; c += 32) {
                float v[32];
                tmem_ld32(ts + c, v);
                wait_ld32(v);
#pragma unroll
                for (int e = 0; e < 32; e += 2) mx = max3(mx, v[e], v[e + 1]);
              }
              mx *= scale;
              // O follows the reference (P V of the tile before has ended).
              float m_new = m;
              if (mx > m + 8.f) {
                m_new = mx;
                alpha = m == -INFINITY ? 0.f : ex2(m - mx);
              }
              if (k > 0 && __any_sync(0xffffffffu, m_new != m)) {
#pragma unroll 1
                for (int c = 0; c < DP; c += 32) {
                  float o[32];
                  tmem_ld32(to + c, o);
                  wait_ld32(o);
#pragma unroll
                  for (int e = 0; e < 32; ++e) o[e] *= alpha;
                  tmem_st32(to + c, o);
                }
              }
              m = m_new;
            }
            // A row that has met no weight yet has no reference either: the lowest
            // number in its place makes the sum of any weight infinite, and is as
            // good as any where all scores are still -inf.
            const float ref = m == -INFINITY ? -FLT_MAX : m;
            float v[2][32];
            add = 0.f;
            tmem_ld32(ts, v[0]);
#pragma unroll
            for (int c = 0; c < kBN; c += 32) {
              wait_ld32(v[(c >> 5) & 1]);
              if (c + 32 < kBN) tmem_ld32(ts + c + 32, v[(c >> 5 & 1) ^ 1]);
              add += weights32<ONE>(v[(c >> 5) & 1], scale, ref, pk + (c >> 1), lo + (ONE ? c >> 1 : 0));
            }
            if (fresh || !__any_sync(0xffffffffu, !(add < 65536.f))) break;
          }
#pragma unroll
          for (int c = 0; c < kBN / 2; c += 16) {
            tmem_st16(ts + c, pk + c);
            if constexpr (ONE) tmem_st16(ts + kBN / 2 + c, lo + c);
          }
          l = l * alpha + add;
          tmem_wait_st();
        }
        if (left < kBN && (one || w == 0)) {
          const uint32_t e = first + 2 * jj + 1;
          ok = warp_wait(&full[e % NS], (e / NS) & 1u, abort_flag);
          if (!ok) break;
          if (r >= left) {
            uint8_t* vrow = smem + L::RING + (e % NS) * L::TILE + r * 128;
#pragma unroll
            for (int h = 0; h < L::HALVES; ++h)
#pragma unroll
              for (int c = 0; c < 8; ++c)
                *reinterpret_cast<uint4*>(vrow + h * L::HALF + c * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_shared();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[w]);
      }
      if (ok && cnt > 0) {
        ok = warp_wait(&o_full[w], oseg & 1u, abort_flag);
        ++oseg;
        tc_fence_after();
      }
      if (!ok) break;
      // Slot of this CTA among those that share the unit.
      const int slot =
          static_cast<int>(blockIdx.x - cta_of(p.units, p.unit_tiles, gridDim.x, sg.unit, 0));
      // The groups' columns and factors: group w writes its own tile, or in the
      // one-tile form half of the columns of f0 O_0 + f1 O_1.
      const bool both = one && n >= 2;
      float f0 = 1.f, f1 = 0.f;
      if (both) {
        // (Maximum, sum) go through the groups' S columns, which are free now.
        tmem_st2(ts, __float_as_uint(m), __float_as_uint(l));
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(merge_full);
        ok = warp_wait(merge_full, mseg & 1u, abort_flag);
        if (!ok) break;
        tc_fence_after();
        uint32_t x0, y0, x1, y1;
        tmem_ld2(tmem + lanes, x0, y0);
        tmem_ld2(tmem + 128 + lanes, x1, y1);
        wait_ld4(x0, y0, x1, y1);
        const float2 a0 = make_float2(__uint_as_float(x0), __uint_as_float(y0));
        const float2 a1 = make_float2(__uint_as_float(x1), __uint_as_float(y1));
        m = fmaxf(a0.x, a1.x);
        f0 = a0.x == -INFINITY ? 0.f : ex2(a0.x - m);
        f1 = a1.x == -INFINITY ? 0.f : ex2(a1.x - m);
        l = a0.y * f0 + a1.y * f1;
      }
      if (warp_live && (both || (one ? w == 0 : group_live))) {
        const int64_t at = (static_cast<int64_t>(g) * s.rows + row) * s.ns + slot;
        // This warp's eighth of the Q tiles is free: every S has been computed.
        constexpr int W = DP / 2;
        RowWriter<W> out;
        out.stage = reinterpret_cast<float*>(smem + L::Q0 + (warp - 4) * (L::TILE / 4));
        out.dst = s.acc + (at - static_cast<int64_t>(lane) * s.ns) * s.D;
        out.pitch = static_cast<int64_t>(s.ns) * s.D;
        out.rows = s.rows - (row - lane);
        out.cols = s.D;
        const uint32_t o0 = tmem + 256 + lanes;
#pragma unroll 1
        for (int c = both ? w * W : 0; c < (both ? (w + 1) * W : DP); c += 32) {
          float o[32];
          tmem_ld32((both ? o0 : to) + c, o);
          if (both) {
            float o1[32];
            tmem_ld32(o0 + 128 + c, o1);
            wait_ld32(o);
            wait_ld32(o1);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = o[e] * f0 + o1[e] * f1;
          } else {
            wait_ld32(o);
          }
          out.put(c, o);
          if ((c + 32) % W == 0) out.flush(c + 32 - W);
        }
        if (row < s.rows && (w == 0 || !both)) {
          float2* dst = reinterpret_cast<float2*>(s.ml) + at;
          dst[0] = make_float2(m, l);
          // The unit's last segment also marks the slots that stay unused.
          if (sg.j0 + n == p.unit_tiles)
            for (int i = slot + 1; i < s.np; ++i) dst[i - slot] = make_float2(-INFINITY, 0.f);
        }
      }
      if (both) {
        // O, Q and ml may be written again once both groups are done with them.
        tc_fence_before();
        mbar_arrive(merge_done);
        ok = warp_wait(merge_done, mseg & 1u, abort_flag);
        tc_fence_after();
        ++mseg;
      } else if (one ? w == 0 : group_live) {
        // The next Q goes over what the group's warps stage their rows in.
        mbar_arrive(&drained[w]);
        ok = warp_wait(&drained[w], dseg & 1u, abort_flag);
        ++dseg;
      }
      first += 2 * n;
    }
    if (!ok) give_up();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512)
                 : "memory");
  }
}

template <int DP, bool ONE>
int launch(const TcParams& p, const b200_kv_pool_t& pool, int ctas, const DeviceInfo& dev,
           cudaStream_t stream) {
  const int smem = TcSmem<DP>::BYTES + 1024;
  if (smem > dev.max_smem_optin)
    return fail(B200_ERR_UNSUPPORTED, "shared prefix: not enough shared memory");
  CUtensorMap tk, tv;
  const uint64_t dims[3] = {static_cast<uint64_t>(pool.head_dim), static_cast<uint64_t>(pool.num_heads),
                            static_cast<uint64_t>(pool.num_layers * pool.num_blocks * pool.block_size)};
  const uint64_t strides[2] = {static_cast<uint64_t>(pool.head_dim * 2),
                               static_cast<uint64_t>(pool.num_heads * pool.head_dim * 2)};
  const uint32_t box[3] = {64u, 1u, static_cast<uint32_t>(p.rbox)};
  int rc = encode_tensor_map(&tk, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, pool.k, dims, strides, box,
                             CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc != B200_OK) return rc;
  rc = encode_tensor_map(&tv, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, pool.v, dims, strides, box,
                         CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc != B200_OK) return rc;
  static std::atomic<int> configured[64];
  if (dev.device >= 64 || !configured[dev.device].load(std::memory_order_acquire)) {
    cudaError_t e = cudaFuncSetAttribute(shared_prefix_tc_kernel<DP, ONE>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(shared prefix)");
    if (dev.device < 64) configured[dev.device].store(1, std::memory_order_release);
  }
  shared_prefix_tc_kernel<DP, ONE><<<static_cast<unsigned>(ctas), kThreads, smem, stream>>>(tk, tv, p);
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? B200_OK : cuda_fail(e, "shared prefix launch");
}

}  // namespace

// One CTA per SM; where the work is less, whole shares of a unit of at least two
// key tiles (a CTA that also has to begin another unit takes 7 us longer); each
// leaves a part that the join reads, so that more than 32 of them are of at least
// four tiles, and there are at most 64 (64 rows of one head, 131072 keys: 53 us,
// with 32 shares 75).
TcSplit shared_tc_split(int64_t rows, int64_t Hkv, int64_t prefix, int num_sms) {
  TcSplit t{};
  t.unit_pairs = static_cast<int>(ceil_div(rows, 2 * kBM));
  t.unit_tiles = static_cast<int>(ceil_div(prefix, kBN));
  t.units = Hkv * t.unit_pairs;
  const int64_t shares = std::max(std::min<int64_t>(ceil_div(t.unit_tiles, 2), 32),
                                  std::min<int64_t>(ceil_div(t.unit_tiles, 4), kPrefixParts));
  t.ctas = static_cast<int>(std::min<int64_t>(num_sms, t.units * shares));
  // The most CTAs that share a unit (an upper bound where the units are many).
  int64_t most = 1;
  if (t.units <= 1024) {
    for (int64_t u = 0; u < t.units; ++u)
      most = std::max(most, cta_of(t.units, t.unit_tiles, t.ctas, u, t.unit_tiles - 1) -
                                cta_of(t.units, t.unit_tiles, t.ctas, u, 0) + 1);
  } else {
    const int64_t least = t.units * (t.unit_tiles + kSegment) / t.ctas;
    most = std::min<int64_t>(ceil_div(t.unit_tiles - 1, least) + 1, t.ctas);
  }
  t.np = static_cast<int>(most);
  return t;
}

int launch_shared_prefix_tc(const SharedParams& s, const b200_kv_pool_t& pool, const TcSplit& t,
                            int zero_count, cudaStream_t stream) {
  DeviceInfo dev;
  int rc = current_device_info(&dev);
  if (rc != B200_OK) return rc;
  TcParams p{};
  p.s = s;
  p.units = t.units;
  p.unit_tiles = t.unit_tiles;
  p.unit_pairs = t.unit_pairs;
  p.rbox = static_cast<int32_t>(std::min<int64_t>(s.S, kBN));
  p.rb_shift = log2i(p.rbox);
  p.q_vec = s.qs2 == 1 && reinterpret_cast<uintptr_t>(s.q) % 16 == 0 && s.qs0 % 8 == 0 && s.qs1 % 8 == 0;
  p.zero_count = zero_count;
  const bool one = s.rows <= kBM;
  if (s.D <= 64)
    return one ? launch<64, true>(p, pool, t.ctas, dev, stream) : launch<64, false>(p, pool, t.ctas, dev, stream);
  return one ? launch<128, true>(p, pool, t.ctas, dev, stream) : launch<128, false>(p, pool, t.ctas, dev, stream);
}

}  // namespace b200
