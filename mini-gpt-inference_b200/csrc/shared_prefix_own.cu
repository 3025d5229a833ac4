// shared_prefix_own.cu -- the sequences' own keys of the shared-prefix decode
// for bf16 pools, and the join with the prefix's parts; and, for few query rows
// and for f16 and f32 queries, the prefix itself, eight rows at a time.
//
// For the rep query rows of one (sequence, key head) this is a matrix-vector
// product per row: bound by the bytes of K and V, each read once for all rep
// rows.  Warp-level matrix products keep the arithmetic out of the way:
//   S^T = K Q^T   (16 keys x 8 rows),   O^T = V^T P^T  (16 d x 8 rows)
// have the keys and the d on the 16-wide side, so that a group of 8 rows
// fills the other; rows from rep on are zero queries whose results are
// dropped.  P^T comes from S^T by an 8x8 transpose within the warp.
//
// What bounds it is the bytes in flight: a row of one head is 256 bytes in a
// place of its own.  Each of the four warps takes every fourth step of 16
// keys, has its own ring of three entries (K of a step, its V, K of the next: 4
// KB each at D = 128) filled by TMA page by page, and needs no other warp until
// the end.  Four CTAs fit an SM, so that one's beginning and join, 6 us for a
// few keys, pass beside the others' loads.  64 sequences of 32 heads with up to
// 1024 own keys (537 MB): 90 us, 6.1 TB/s; 256 of up to 64 keys, behind 256, 99
// us in all.  With entries of K and V, two to a warp, and three CTAs 89 and 116
// us; with three of them, and two CTAs, the first 95 us; with the operands loaded
// straight into registers, one step a warp, 213 us.  (The prefix's parts, which
// are long and few, keep the larger entries: a wait less in each step.)  f16 and
// f32 queries cost little more, and far less than f32 arithmetic: 64 sequences of
// 8 x 4 heads behind 4096 keys 80 and 90 us (element kernels 219), 4 behind 32768
// 42 and 45 (185).
#include <algorithm>
#include <atomic>

#include "common.cuh"
#include "host_util.h"
#include "kernels.h"
#include "shared_prefix.cuh"
#include "tcgen05.cuh"

namespace b200 {
namespace {

constexpr int kWarps = 4;
constexpr int kStep = 16;      // keys a warp takes at a time
constexpr int kAhead = 8;      // parts of a row that the join loads together (4 and 16: 1 to 5 % slower at
                               // many parts, and at many short joins)
constexpr int kMaxSlots = kPrefixParts + kOwnParts + kWarps;  // parts of a row, and the warps' states

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// c += a b: 16 x 16 by 16 x 8, bf16 with f32 sums.
__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void ldmatrix4(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

struct OwnParams {
  SharedParams s;
  int32_t rbox, rb_shift;  // rows per TMA box: min(S, 16)
  int32_t q_vec;           // 4-byte access to pairs of q is legal
  int32_t out_vec;         // 8-byte access to four elements of bf16 out is legal
  int32_t zero_count;      // PREFIX: counters to clear
};

template <int DP, bool PREFIX, int QP>
struct OwnSmem {
  static constexpr int HALVES = DP / 64;
  static constexpr int HALF = kStep * 128;        // 16 keys x 64 d
  static constexpr int TILE = HALVES * HALF;      // K or V of a step
  // Ring entries: K or V of a step where three of them leave room for four CTAs on
  // an SM (own keys, where registers do too), else both, twice (see above).
  static constexpr bool SPLIT = !PREFIX && QP <= 2;
  static constexpr int ENTRY = SPLIT ? TILE : 2 * TILE;
  static constexpr int ENTRIES = (SPLIT ? 3 : 2) * (DP == 128 ? 1 : 2);
  static constexpr int RING = kWarps * ENTRIES * ENTRY;
  static constexpr int R = kOwnRows;
  static constexpr int LD = DP + 4;               // 2 LD = 8 mod 32: no bank is hit twice
  static constexpr int MERGE = kWarps * R * LD * 4;  // the warps' O, over the ring
  static constexpr int BAR = RING > MERGE ? RING : MERGE;
  static constexpr int ML = BAR + kWarps * ENTRIES * 8;  // float2 [kMaxSlots][R]
  static constexpr int BYTES = ML + kMaxSlots * R * 8 + 16;
  static_assert(TILE % 1024 == 0, "swizzled tiles start on 1024 bytes");
};

// DP: head dimension rounded up to 64 or 128.
// PREFIX: the keys are a part of the prefix's, the rows all sequences'.
// QP: bf16 pieces that a query element is the sum of: 1 for bf16, 2 for f16 (11
// bits), 3 for f32 (24 bits), in all its bits (and 2^-30 of it at most where a
// piece would be zero).  A piece is another product, and there is time for them.  The weights take part in as many pieces, and at least in two:
// what is left of them is at most 2^-16, with three 2^-24.
template <int DP, bool PREFIX, int QP>
__global__ void __launch_bounds__(kWarps * 32)
    shared_own_mma_kernel(const __grid_constant__ CUtensorMap tmk,
                          const __grid_constant__ CUtensorMap tmv, const __grid_constant__ OwnParams op) {
  using L = OwnSmem<DP, PREFIX, QP>;
  constexpr int NS = L::ENTRIES, R = L::R, PP = QP == 3 ? 3 : 2;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const SharedParams& p = op.s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int gq = lane >> 2, t = lane & 3;  // fragment row and column pair

  // Heads fastest: CTAs that run together read neighbouring columns of the
  // same pages.
  int64_t idx = blockIdx.x;
  const int g = static_cast<int>(idx % p.Hkv);
  idx /= p.Hkv;
  const int chunk = static_cast<int>(idx % p.row_chunks);
  idx /= p.row_chunks;
  const int split = static_cast<int>(PREFIX ? idx : idx % p.own_splits);
  const int b = static_cast<int>(PREFIX ? 0 : idx / p.own_splits);
  const int row0 = (PREFIX ? 0 : b * p.rep) + chunk * R;
  const int nrows = min(R, (PREFIX ? p.rows : p.rep) - chunk * R);
  const int head0 = g * p.rep + chunk * R;  // own keys only
  if constexpr (PREFIX) {
    let_next_start();
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * (kWarps * 32) + threadIdx.x; i < op.zero_count;
         i += static_cast<int64_t>(gridDim.x) * (kWarps * 32))
      p.cnt[i] = 0;  // of the own-key kernel
  }
  const int64_t ctx = PREFIX ? p.prefix : load_index(p.lens, b * p.len_stride, p.lens_i64);
  if (!PREFIX && (ctx < 1 || ctx < p.prefix || ctx > p.table_width * p.S)) {
    if (split == 0) {
      if (threadIdx.x == 0) report(p.status, B200_DEV_BAD_LENGTH);
      if (p.out == p.q) wait_for_previous();  // it reads these rows
      for (int i = threadIdx.x; i < nrows * p.D; i += kWarps * 32)
        store_elem(p.out, b * p.os0 + (head0 + i / p.D) * p.os1 + (i % p.D) * p.os2, p.out_dtype, 0.f);
    }
    end_after_previous();
    return;
  }
  // Steps lie on multiples of 16 positions, so that no step's box leaves its
  // page; the keys outside [lo, hi) of the first and last one are masked.
  int64_t k0, hi, lo;
  int parts = 1;
  if constexpr (PREFIX) {
    lo = k0 = static_cast<int64_t>(split) * p.prefix_per;
    hi = min(p.prefix, k0 + p.prefix_per);
  } else {
    const int64_t origin = p.prefix & ~int64_t(kStep - 1);
    parts = own_range(p, ctx > p.prefix ? ctx - origin : 0, split, &k0, &hi);
    if (split >= parts) {
      end_after_previous();
      return;
    }
    k0 += origin;
    hi += origin;
    lo = max(k0, p.prefix);
  }
  const int steps = static_cast<int>((hi - k0 + kStep - 1) / kStep);
  const int mine = (steps - warp + kWarps - 1) / kWarps;  // of this warp: warp, warp + 4, ...

  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::BAR) + warp * NS;
  uint8_t* ring = smem + warp * (NS * L::ENTRY);
  if (lane < NS) mbar_init(&full[lane], 1);
  fence_mbar_init();
  __syncwarp();

  // Boxes of step n: nb of them, box i holding keys first + i * rbox.  A lane
  // keeps the pool row of box (lane % nb) of step (batch + lane / nb).
  const int nb = kStep >> op.rb_shift;
  const int per_batch = 32 / nb;
  auto lookup = [&](int n) -> int {  // for lane's step n + lane / nb
    const int64_t key = k0 + static_cast<int64_t>(warp + kWarps * (n + lane / nb)) * kStep +
                        ((lane % nb) << op.rb_shift);
    if (n + lane / nb >= mine || key >= hi || key + op.rbox <= lo) return -1;
    int64_t e = PREFIX ? load_index(p.prefix_table, (key >> p.s_shift) * p.pt_stride, p.pt_i64)
                       : load_index(p.tables, b * p.ts0 + (key >> p.s_shift) * p.ts1, p.tables_i64);
    if (e < 0 || e >= p.P) {
      report(p.status, B200_DEV_BAD_BLOCK);
      e = 0;  // an in-bounds page; the status word tells
    }
    return static_cast<int>(p.layer_row0 + e * p.S + (key & (p.S - 1)));
  };
  int rows = lookup(0);
  int rows_next = mine > per_batch ? lookup(per_batch) : -1;
  int batch = 0;
  constexpr bool split_kv = L::SPLIT;
  auto issue = [&](int e) {  // entry e: K (even) or V of step e / 2, or step e
    const int n = split_kv ? e >> 1 : e, st = e % NS;
    if (n >= batch + per_batch) {
      batch += per_batch;
      rows = rows_next;
      rows_next = batch + per_batch < mine ? lookup(batch + per_batch) : -1;
    }
    const int box = lane % nb, rest = lane / nb;  // of this lane
    const int half = rest % L::HALVES, kv = split_kv ? e & 1 : rest / L::HALVES;
    const int row = __shfl_sync(0xffffffffu, rows, (n - batch) * nb + box);
    const unsigned there = __ballot_sync(0xffffffffu, lane < nb && row >= 0);
    if (lane == 0)
      mbar_arrive_expect_tx(&full[st], static_cast<uint32_t>(__popc(there) * (L::ENTRY / L::HALF) * op.rbox * 128));
    __syncwarp();
    if (rest < L::ENTRY / L::HALF && row >= 0)
      tma_load_3d(ring + st * L::ENTRY + rest * L::HALF + box * op.rbox * 128, kv == 0 ? &tmk : &tmv, &full[st],
                  half * 64, g, row);
  };
  auto arrived = [&](int e) {
    return __all_sync(0xffffffffu, mbar_wait(&full[e % NS], static_cast<uint32_t>(e / NS) & 1u)) != 0;
  };
  const int entries = split_kv ? 2 * mine : mine;
  int issued = min(entries, NS);
  for (int n = 0; n < issued; ++n) issue(n);

  // Query fragments: row gq, d = 16 i + 2t + {0, 1} and + 8.
  uint32_t qf[QP][DP / 16][2];
#pragma unroll
  for (int i = 0; i < DP / 16; ++i)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int r = gq, d = 16 * i + 2 * t + 8 * u;
#pragma unroll
      for (int c = 0; c < QP; ++c) qf[c][i][u] = 0;
      if (r < nrows && d < p.D) {
        const int seq = PREFIX ? (row0 + r) / p.rep : b;
        const int head = PREFIX ? g * p.rep + (row0 + r) - seq * p.rep : head0 + r;
        const int64_t at = seq * p.qs0 + head * p.qs1 + d * p.qs2;
        if (QP == 1 && op.q_vec) {
          qf[0][i][u] = *reinterpret_cast<const uint32_t*>(static_cast<const __nv_bfloat16*>(p.q) + at);
        } else {
          constexpr int type = QP == 1 ? B200_DTYPE_BF16 : QP == 2 ? B200_DTYPE_F16 : B200_DTYPE_F32;
          const float x = load_elem(p.q, at, type), y = load_elem(p.q, at + p.qs2, type);
          float rx = x, ry = y;  // what the pieces so far leave
#pragma unroll
          for (int c = 0; c < QP; ++c) {
            qf[c][i][u] = chop_bf16(rx, ry);
            const float2 f = bf16x2_to_float2(qf[c][i][u]);
            rx = fmaf(x, kKeepSign, rx - f.x), ry = fmaf(y, kKeepSign, ry - f.y);
          }
        }
      }
    }

  // Row 2t + u: m[u] (the same in its 8 lanes) and this lane's l;
  // o[i]: d = 16 i + gq (+ 8) of rows 2t, 2t + 1.
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[DP / 16][4];
#pragma unroll
  for (int i = 0; i < DP / 16; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
  // Byte offsets of this lane's ldmatrix row and its chunk's swizzle.  K: keys
  // (lane & 15), chunks 2 i + (lane >> 4); V: keys (lane & 7) + 8 (lane >> 4),
  // chunks 2 i + (lane >> 3 & 1).
  const uint32_t k_row = (lane & 15) * 128, k_hi = lane >> 4;
  const uint32_t v_row = ((lane & 7) + 8 * (lane >> 4)) * 128, v_hi = (lane >> 3) & 1;
  const uint32_t sw = lane & 7;

  bool ok = true;
  for (int n = 0; n < mine; ++n) {
    const int e = split_kv ? 2 * n : n;
    ok = arrived(e);
    if (!ok) break;
    const uint32_t kt = smem_u32(ring + e % NS * L::ENTRY);
    const uint32_t vt = split_kv ? smem_u32(ring + (e + 1) % NS * L::ENTRY) : kt + L::TILE;
    float s[2][4];  // two chains of products
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e >> 2][e & 3] = 0.f;
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) {
      uint32_t a[4];
      const uint32_t ch = (2 * i + k_hi) & 7;
      ldmatrix4(a, kt + (i / 4) * L::HALF + k_row + ((ch ^ sw) << 4));
#pragma unroll
      for (int w = 0; w < QP; ++w) mma16816(s[i & 1], a, qf[w][i][0], qf[w][i][1]);
    }
    if constexpr (split_kv) {
      __syncwarp();  // every lane has read K
      if (issued < entries) issue(issued++);
    }
    const int64_t key = k0 + static_cast<int64_t>(warp + kWarps * n) * kStep;
    const bool edge = key < lo || key + kStep > hi;
    const bool in0 = !edge || (key + gq >= lo && key + gq < hi);
    const bool in1 = !edge || (key + gq + 8 >= lo && key + gq + 8 < hi);
    uint32_t pb[PP][2];  // the weights in bf16, and what that left
    float x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      x[e] = (e < 2 ? in0 : in1) ? (s[0][e] + s[1][e]) * p.qscale : -INFINITY;
    const float mx0 = fmaxf(x[0], x[2]), mx1 = fmaxf(x[1], x[3]);
    // The reference point moves only when a score exceeds it by more than
    // 2^8: weights stay below 2^8 and l and o stay exact relative to it.
    if (__any_sync(0xffffffffu, mx0 > m[0] + 8.f || mx1 > m[1] + 8.f)) {
      float r0 = mx0, r1 = mx1;
#pragma unroll
      for (int w = 4; w <= 16; w <<= 1) {
        r0 = fmaxf(r0, __shfl_xor_sync(0xffffffffu, r0, w));
        r1 = fmaxf(r1, __shfl_xor_sync(0xffffffffu, r1, w));
      }
      r0 = fmaxf(m[0], r0);
      r1 = fmaxf(m[1], r1);
      const float a0 = m[0] == -INFINITY ? 0.f : ex2(m[0] - r0);
      const float a1 = m[1] == -INFINITY ? 0.f : ex2(m[1] - r1);
      m[0] = r0;
      m[1] = r1;
      l[0] *= a0;
      l[1] *= a1;
#pragma unroll
      for (int i = 0; i < DP / 16; ++i) {
        o[i][0] *= a0;
        o[i][1] *= a1;
        o[i][2] *= a0;
        o[i][3] *= a1;
      }
    }
    const float ref0 = m[0] == -INFINITY ? 0.f : m[0];
    const float ref1 = m[1] == -INFINITY ? 0.f : m[1];
    const float p0 = ex2(x[0] - ref0), p1 = ex2(x[1] - ref1);
    const float p2 = ex2(x[2] - ref0), p3 = ex2(x[3] - ref1);
    l[0] += p0 + p2;
    l[1] += p1 + p3;
    float r0 = p0, r1 = p1, r2 = p2, r3 = p3;  // what the pieces so far leave
#pragma unroll
    for (int w = 0; w < PP; ++w) {
      const bool last = w == PP - 1;
      const uint32_t h0 = last ? pack_bf16(r0, r1) : chop_bf16(r0, r1);
      const uint32_t h1 = last ? pack_bf16(r2, r3) : chop_bf16(r2, r3);
      pb[w][0] = transpose8x8(h0);
      pb[w][1] = transpose8x8(h1);
      const float2 f0 = bf16x2_to_float2(h0), f1 = bf16x2_to_float2(h1);
      r0 = fmaf(p0, kKeepSign, r0 - f0.x), r1 = fmaf(p1, kKeepSign, r1 - f0.y);
      r2 = fmaf(p2, kKeepSign, r2 - f1.x), r3 = fmaf(p3, kKeepSign, r3 - f1.y);
    }
    // V rows of masked keys may hold anything, and 0 * NaN is NaN.
    uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;
    if (edge) {
      auto in = [&](int j) { return key + j >= lo && key + j < hi; };
      keep0 = (in(2 * t) ? 0xffffu : 0u) | (in(2 * t + 1) ? 0xffff0000u : 0u);
      keep1 = (in(2 * t + 8) ? 0xffffu : 0u) | (in(2 * t + 9) ? 0xffff0000u : 0u);
    }
    if constexpr (split_kv) {
      ok = arrived(e + 1);
      if (!ok) break;
    }
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) {
      uint32_t a[4];
      const uint32_t ch = (2 * i + v_hi) & 7;
      ldmatrix4_trans(a, vt + (i / 4) * L::HALF + v_row + ((ch ^ sw) << 4));
      a[0] &= keep0;
      a[1] &= keep0;
      a[2] &= keep1;
      a[3] &= keep1;
#pragma unroll
      for (int w = 0; w < PP; ++w) mma16816(o[i], a, pb[w][0], pb[w][1]);
    }
    __syncwarp();  // every lane has read V, or both
    if (issued < entries) issue(issued++);
  }
  if (!ok) {
    if (lane == 0) report(p.status, B200_DEV_WAIT_TIMEOUT);
    for (int e = max(0, issued - NS); e < issued; ++e) mbar_wait(&full[e % NS], static_cast<uint32_t>(e / NS) & 1u);
  }

  // Whole sums of the rows' weights; the warps' states meet in shared memory.
  __syncthreads();  // the ring is free
  float* s_o = reinterpret_cast<float*>(smem);
  float2* s_ml = reinterpret_cast<float2*>(smem + L::ML);
  int* s_last = reinterpret_cast<int*>(smem + L::ML + kMaxSlots * R * 8);
#pragma unroll
  for (int u = 0; u < 2; ++u) {
#pragma unroll
    for (int w = 4; w <= 16; w <<= 1) l[u] += __shfl_xor_sync(0xffffffffu, l[u], w);
    const int r = 2 * t + u;
    if (gq == 0) s_ml[warp * R + r] = make_float2(m[u], l[u]);
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) {
      s_o[(warp * R + r) * L::LD + 16 * i + gq] = o[i][u];
      s_o[(warp * R + r) * L::LD + 16 * i + gq + 8] = o[i][u + 2];
    }
  }
  __syncthreads();

  // Nothing so far, nor this part's way to its slot, comes from the prefix's
  // kernel, whose end this kernel overlaps; its parts, and the counters that it
  // cleared, do.
  const int64_t slot_row = (static_cast<int64_t>(g) * p.rows + row0) * p.ns;
  int warps = kWarps, slots = p.np;  // what is joined: the warps' states, slots of the workspace
  if (PREFIX || parts > 1) {
    // This part goes to its slot; the last one to arrive joins all.
    for (int i = threadIdx.x; i < nrows * (p.D / 4); i += kWarps * 32) {
      const int r = i / (p.D / 4), d = (i % (p.D / 4)) * 4;
      float M = -INFINITY, sum = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) M = fmaxf(M, s_ml[w * R + r].x);
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float2 ml = s_ml[w * R + r];
        const float f = ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : 1.f) : ex2(ml.x - M);
        const float4 v = *reinterpret_cast<const float4*>(s_o + (w * R + r) * L::LD + d);
        sum = fmaf(f, ml.y, sum);
        a.x = fmaf(f, v.x, a.x), a.y = fmaf(f, v.y, a.y), a.z = fmaf(f, v.z, a.z), a.w = fmaf(f, v.w, a.w);
      }
      const int64_t at = slot_row + static_cast<int64_t>(r) * p.ns + (PREFIX ? split : p.np + split);
      *reinterpret_cast<float4*>(p.acc + at * p.D + d) = a;
      if (d == 0) *reinterpret_cast<float2*>(p.ml + at * 2) = make_float2(M, sum);
    }
    if constexpr (PREFIX) return;
    wait_for_previous();
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
      const int64_t unit = (static_cast<int64_t>(b) * p.Hkv + g) * p.row_chunks + chunk;
      *s_last = atomicAdd(&p.cnt[unit], 1) == parts - 1;
    }
    __syncthreads();
    if (!*s_last) return;
    __threadfence();
    warps = 0;
    slots = p.np + parts;
  } else {
    wait_for_previous();
  }

  // Two accesses to memory, one behind the other, would be most of a small call's
  // join, so a thread's first parts are on their way before their factors are
  // known (slots that stay unused hold anything: their factor is 0).
  const int items = nrows * (p.D / 4);
  float4 v[kAhead];
  auto fetch = [&](int i, int j0) {
    const float* acc = p.acc + (slot_row + static_cast<int64_t>(i / (p.D / 4)) * p.ns + j0) * p.D + (i % (p.D / 4)) * 4;
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (j0 + k < slots) v[k] = __ldcg(reinterpret_cast<const float4*>(acc + static_cast<int64_t>(k) * p.D));
  };
  if (threadIdx.x < items) fetch(threadIdx.x, 0);

  // Factors 2^(m - M) / L of every part of every row, a warp per row.
  const int total = warps + slots;
  for (int i = threadIdx.x; i < slots * nrows; i += kWarps * 32) {
    const int j = i / nrows, r = i % nrows;
    s_ml[(warps + j) * R + r] = __ldcg(
        reinterpret_cast<const float2*>(p.ml + (slot_row + static_cast<int64_t>(r) * p.ns + j) * 2));
  }
  __syncthreads();
  for (int r = warp; r < nrows; r += kWarps) {
    float M = -INFINITY;
    for (int j = lane; j < total; j += 32) M = fmaxf(M, s_ml[j * R + r].x);
#pragma unroll
    for (int w = 16; w >= 1; w >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, w));
    float sum = 0.f;
    for (int j = lane; j < total; j += 32) {
      const float2 ml = s_ml[j * R + r];
      // An empty part (no key, or a slot that stays unused) has no factor.
      const float f = ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : 1.f) : ex2(ml.x - M);
      s_ml[j * R + r].x = f;
      sum = fmaf(f, ml.y, sum);
    }
#pragma unroll
    for (int w = 16; w >= 1; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
    const float inv = 1.0f / sum;
    for (int j = lane; j < total; j += 32) s_ml[j * R + r].x *= inv;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < items; i += kWarps * 32) {
    const int r = i / (p.D / 4), d = (i % (p.D / 4)) * 4;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](float f, const float4& x) {
      a.x = fmaf(f, x.x, a.x), a.y = fmaf(f, x.y, a.y), a.z = fmaf(f, x.z, a.z), a.w = fmaf(f, x.w, a.w);
    };
    for (int j = 0; j < warps; ++j)
      add(s_ml[j * R + r].x, *reinterpret_cast<const float4*>(s_o + (j * R + r) * L::LD + d));
    for (int j0 = 0; j0 < slots; j0 += kAhead) {
      if (i != threadIdx.x || j0 > 0) fetch(i, j0);
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const float f = j0 + k < slots ? s_ml[(warps + j0 + k) * R + r].x : 0.f;
        if (f != 0.f) add(f, v[k]);
      }
    }
    const int64_t at = b * p.os0 + (head0 + r) * p.os1 + d * p.os2;
    if (op.out_vec) {
      *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.out) + at) =
          make_uint2(pack_bf16(a.x, a.y), pack_bf16(a.z, a.w));
    } else {
      store_elem(p.out, at, p.out_dtype, a.x);
      store_elem(p.out, at + p.os2, p.out_dtype, a.y);
      store_elem(p.out, at + 2 * p.os2, p.out_dtype, a.z);
      store_elem(p.out, at + 3 * p.os2, p.out_dtype, a.w);
    }
  }
}

template <int DP, bool PREFIX, int QP>
int launch_one(const OwnParams& op, const b200_kv_pool_t& pool, const DeviceInfo& dev, bool overlap,
           cudaStream_t stream) {
  const SharedParams& p = op.s;
  const int64_t grid = static_cast<int64_t>(PREFIX ? p.np : p.B * p.own_splits) * p.row_chunks * p.Hkv;
  const int smem = OwnSmem<DP, PREFIX, QP>::BYTES + 1024;
  CUtensorMap tk, tv;
  const uint64_t dims[3] = {static_cast<uint64_t>(pool.head_dim), static_cast<uint64_t>(pool.num_heads),
                            static_cast<uint64_t>(pool.num_layers * pool.num_blocks * pool.block_size)};
  const uint64_t strides[2] = {static_cast<uint64_t>(pool.head_dim * 2),
                               static_cast<uint64_t>(pool.num_heads * pool.head_dim * 2)};
  const uint32_t box[3] = {64u, 1u, static_cast<uint32_t>(op.rbox)};
  int rc = encode_tensor_map(&tk, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, pool.k, dims, strides, box,
                             CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc != B200_OK) return rc;
  rc = encode_tensor_map(&tv, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, pool.v, dims, strides, box,
                         CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc != B200_OK) return rc;
  auto kern = shared_own_mma_kernel<DP, PREFIX, QP>;
  static std::atomic<int> configured[64];
  if (dev.device >= 64 || !configured[dev.device].load(std::memory_order_acquire)) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(shared prefix)");
    if (dev.device < 64) configured[dev.device].store(1, std::memory_order_release);
  }
  return launch_own(kern, grid, kWarps * 32, smem, stream, overlap, tk, tv, op);
}

template <bool PREFIX>
int launch(const OwnParams& op, const b200_kv_pool_t& pool, const DeviceInfo& dev, bool overlap,
           cudaStream_t stream) {
  const bool d64 = op.s.D <= 64;
  if (op.s.q_dtype == B200_DTYPE_F16)
    return d64 ? launch_one<64, PREFIX, 2>(op, pool, dev, overlap, stream)
               : launch_one<128, PREFIX, 2>(op, pool, dev, overlap, stream);
  if (op.s.q_dtype == B200_DTYPE_F32)
    return d64 ? launch_one<64, PREFIX, 3>(op, pool, dev, overlap, stream)
               : launch_one<128, PREFIX, 3>(op, pool, dev, overlap, stream);
  return d64 ? launch_one<64, PREFIX, 1>(op, pool, dev, overlap, stream)
             : launch_one<128, PREFIX, 1>(op, pool, dev, overlap, stream);
}

bool aligned(const void* p, int64_t s0, int64_t s1, int64_t s2, int bytes) {
  return s2 == 1 && reinterpret_cast<uintptr_t>(p) % bytes == 0 && s0 % (bytes / 2) == 0 &&
         s1 % (bytes / 2) == 0;
}

OwnParams own_params(const SharedParams& p, int zero_count) {
  OwnParams op;
  op.s = p;
  op.rbox = static_cast<int32_t>(std::min<int64_t>(p.S, kStep));
  op.rb_shift = log2i(op.rbox);
  op.q_vec = aligned(p.q, p.qs0, p.qs1, p.qs2, 4);
  op.out_vec = p.out_dtype == B200_DTYPE_BF16 && aligned(p.out, p.os0, p.os1, p.os2, 8);
  op.zero_count = zero_count;
  return op;
}

}  // namespace

int launch_shared_own_mma(const SharedParams& p, const b200_kv_pool_t& pool, bool overlap,
                          cudaStream_t stream) {
  DeviceInfo dev;
  int rc = current_device_info(&dev);
  if (rc != B200_OK) return rc;
  return launch<false>(own_params(p, 0), pool, dev, overlap, stream);
}

int launch_shared_prefix_mma(const SharedParams& p, const b200_kv_pool_t& pool, int zero_count,
                             cudaStream_t stream) {
  DeviceInfo dev;
  int rc = current_device_info(&dev);
  if (rc != B200_OK) return rc;
  OwnParams op = own_params(p, zero_count);
  op.s.row_chunks = static_cast<int32_t>(ceil_div(p.rows, kOwnRows));
  return launch<true>(op, pool, dev, false, stream);
}

}  // namespace b200
