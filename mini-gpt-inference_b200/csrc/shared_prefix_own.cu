// shared_prefix_own.cu -- the sequences' own keys of the shared-prefix decode
// for bf16 pools and queries, and the join with the prefix's parts.
//
// For the rep query rows of one (sequence, key head) this is a matrix-vector
// product per row: bound by the bytes of K and V, each read once for all rep
// rows.  Warp-level matrix products keep the arithmetic out of the way with
// few instructions per byte, and are arranged so that every operand comes from
// global memory straight into registers, 16 bytes a load, with no staging:
//   S^T = K Q^T   (16 keys x 8 rows): the sum over d may run in any order, so
//       a lane takes 16-byte chunks of a key's row as they lie; the query's
//       fragment holds the same chunks.
//   O^T = V^T P^T (16 d x 8 rows): a lane loads the same 8 d of four keys and
//       pairs them up with byte permutes; the rows of an O^T tile are those d.
// P^T comes from S^T by an 8x8 transpose within the warp.  Rows from rep on
// are zero queries whose results are dropped.
//
// A warp works on 16 keys at a time, four warps side by side; the next step's
// K is requested when this step's scores are done, its V when the outputs
// are, its table entries a step earlier, so that loads are in flight all the
// time (8 KB a warp at D = 128).
#include <algorithm>

#include "common.cuh"
#include "host_util.h"
#include "kernels.h"
#include "shared_prefix.cuh"
#include "tcgen05.cuh"

namespace b200 {
namespace {

constexpr int kWarps = 4;
constexpr int kStep = 16;  // keys a warp takes at a time

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// c += a b: 16 x 16 by 16 x 8, bf16 with f32 sums.
__device__ __forceinline__ void mma16816(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ uint4 load_chunk(const uint8_t* p, bool ok) {
  return ok ? __ldg(reinterpret_cast<const uint4*>(p)) : make_uint4(0, 0, 0, 0);
}

struct OwnParams {
  SharedParams s;
  int32_t q_vec, out_vec;  // 16-byte access to rows of q / bf16 out is legal
};

// NQ groups of 8 query rows; DP: head dimension rounded up to 64 or 128.
template <int DP, int NQ>
__global__ void __launch_bounds__(kWarps * 32, NQ == 1 ? 3 : 2)
    shared_own_mma_kernel(const __grid_constant__ OwnParams op) {
  constexpr int KC = DP / 32;  // K chunks per lane and row
  constexpr int VH = DP / 64;  // V chunks per lane and key
  constexpr int R = 8 * NQ;
  constexpr int LD = DP + 8;
  __shared__ float s_o[kWarps][R][LD];
  __shared__ float s_m[kWarps][R], s_l[kWarps][R];
  __shared__ int s_last;
  const SharedParams& p = op.s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int gq = lane >> 2, t = lane & 3;  // fragment row and column pair

  // Heads fastest, then parts: CTAs that run together read neighbouring
  // columns of the same pages.
  int64_t idx = blockIdx.x;
  const int g = static_cast<int>(idx % p.Hkv);
  idx /= p.Hkv;
  const int chunk = static_cast<int>(idx % p.row_chunks);
  idx /= p.row_chunks;
  const int split = static_cast<int>(idx % p.own_splits);
  const int b = static_cast<int>(idx / p.own_splits);
  const int row0 = b * p.rep + chunk * R;
  const int nrows = min(R, p.rep - chunk * R);
  const int64_t ctx = load_index(p.lens, b * p.len_stride, p.lens_i64);
  if (ctx < 1 || ctx < p.prefix || ctx > p.table_width * p.S) {
    if (split == 0) {
      if (threadIdx.x == 0) report(p.status, B200_DEV_BAD_LENGTH);
      for (int i = threadIdx.x; i < nrows * p.D; i += kWarps * 32)
        store_elem(p.out, b * p.os0 + (g * p.rep + chunk * R + i / p.D) * p.os1 + (i % p.D) * p.os2,
                   p.out_dtype, 0.f);
    }
    return;
  }
  int64_t k0, k1;
  const int parts = own_range(p, ctx - p.prefix, split, &k0, &k1);
  if (split >= parts) return;
  k0 += p.prefix;
  k1 += p.prefix;

  // Table entry -> pool row of key base + lane (lanes 0..15), -1 past the end.
  auto entry = [&](int64_t base) -> int64_t {
    const int64_t key = base + lane;
    if (lane >= kStep || key >= k1) return -1;
    return load_index(p.tables, b * p.ts0 + (key >> p.s_shift) * p.ts1, p.tables_i64);
  };
  auto row_of = [&](int64_t base, int64_t e) -> int {
    const int64_t key = base + lane;
    if (lane >= kStep || key >= k1) return -1;
    if (e < 0 || e >= p.P) {
      report(p.status, B200_DEV_BAD_BLOCK);
      e = 0;  // an in-bounds page; the status word tells
    }
    return static_cast<int>(p.layer_row0 + e * p.S + (key & (p.S - 1)));
  };
  const int64_t row_bytes = static_cast<int64_t>(p.Hkv) * p.D * 2;
  const uint8_t* kbase = static_cast<const uint8_t*>(p.k_pool) + static_cast<int64_t>(g) * p.D * 2;
  const uint8_t* vbase = static_cast<const uint8_t*>(p.v_pool) + static_cast<int64_t>(g) * p.D * 2;
  const int nchunks = p.D / 8;

  uint4 kf[2][KC], vf[4][VH];
  auto load_k = [&](int row) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = __shfl_sync(0xffffffffu, row, gq + 8 * h);
      const uint8_t* src = kbase + r * row_bytes + t * 16;
#pragma unroll
      for (int i = 0; i < KC; ++i) kf[h][i] = load_chunk(src + i * 64, r >= 0 && t + 4 * i < nchunks);
    }
  };
  auto load_v = [&](int row) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = __shfl_sync(0xffffffffu, row, 2 * t + (j & 1) + 8 * (j >> 1));
      const uint8_t* src = vbase + r * row_bytes + gq * 16;
#pragma unroll
      for (int h = 0; h < VH; ++h) vf[j][h] = load_chunk(src + h * 128, r >= 0 && gq + 8 * h < nchunks);
    }
  };

  int64_t base = k0 + warp * kStep;
  int row = -1;
  int64_t e_next = -1;
  if (base < k1) {
    row = row_of(base, entry(base));
    load_k(row);
    load_v(row);
    e_next = entry(base + kWarps * kStep);
  }

  // Query fragments: row 8n + gq, the chunks t + 4i.
  uint4 qf[NQ][KC];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int r = 8 * n + gq;
#pragma unroll
    for (int i = 0; i < KC; ++i) {
      const int c = t + 4 * i;
      qf[n][i] = make_uint4(0, 0, 0, 0);
      if (r < nrows && c < nchunks) {
        const int64_t at = b * p.qs0 + (g * p.rep + chunk * R + r) * p.qs1 + c * 8 * p.qs2;
        const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(p.q);
        if (op.q_vec) {
          qf[n][i] = *reinterpret_cast<const uint4*>(q + at);
        } else {
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const __nv_bfloat162 x = __halves2bfloat162(q[at + 2 * e * p.qs2], q[at + (2 * e + 1) * p.qs2]);
            w[e] = *reinterpret_cast<const uint32_t*>(&x);
          }
          qf[n][i] = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
    }
  }

  // Row 8n + 2t + u: m[n][u] (the same in its 8 lanes) and this lane's l.
  float m[NQ][2], l[NQ][2], o[NQ][VH][4][4];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    m[n][0] = m[n][1] = -INFINITY;
    l[n][0] = l[n][1] = 0.f;
#pragma unroll
    for (int h = 0; h < VH; ++h)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][h][j][e] = 0.f;
  }
  // New maxima mn for the rows of group n: l and o follow.
  auto rescale = [&](int n, float mn0, float mn1) {
    const float a0 = m[n][0] == -INFINITY ? 0.f : ex2(m[n][0] - mn0);
    const float a1 = m[n][1] == -INFINITY ? 0.f : ex2(m[n][1] - mn1);
    m[n][0] = mn0;
    m[n][1] = mn1;
    l[n][0] *= a0;
    l[n][1] *= a1;
#pragma unroll
    for (int h = 0; h < VH; ++h)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        o[n][h][j][0] *= a0;
        o[n][h][j][1] *= a1;
        o[n][h][j][2] *= a0;
        o[n][h][j][3] *= a1;
      }
  };

  for (; base < k1; base += kWarps * kStep) {
    float s[NQ][4];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
#pragma unroll
      for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
#pragma unroll
      for (int i = 0; i < KC; ++i) {
        mma16816(s[n], kf[0][i].x, kf[1][i].x, kf[0][i].y, kf[1][i].y, qf[n][i].x, qf[n][i].y);
        mma16816(s[n], kf[0][i].z, kf[1][i].z, kf[0][i].w, kf[1][i].w, qf[n][i].z, qf[n][i].w);
      }
    }
    const int64_t next = base + kWarps * kStep;
    int row_next = -1;
    if (next < k1) {
      row_next = row_of(next, e_next);
      load_k(row_next);
      e_next = entry(next + kWarps * kStep);
    }
    const bool in0 = base + gq < k1, in1 = base + gq + 8 < k1;
    uint32_t pb[NQ][2];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = (e < 2 ? in0 : in1) ? s[n][e] * p.qscale : -INFINITY;
      const float mx0 = fmaxf(x[0], x[2]), mx1 = fmaxf(x[1], x[3]);
      // The reference point moves only when a score exceeds it by more than
      // 2^8: weights stay below 2^8 and the parts' exact l and o follow it.
      if (__any_sync(0xffffffffu, mx0 > m[n][0] + 8.f || mx1 > m[n][1] + 8.f)) {
        float r0 = mx0, r1 = mx1;
#pragma unroll
        for (int w = 4; w <= 16; w <<= 1) {
          r0 = fmaxf(r0, __shfl_xor_sync(0xffffffffu, r0, w));
          r1 = fmaxf(r1, __shfl_xor_sync(0xffffffffu, r1, w));
        }
        rescale(n, fmaxf(m[n][0], r0), fmaxf(m[n][1], r1));
      }
      const float ref0 = m[n][0] == -INFINITY ? 0.f : m[n][0];
      const float ref1 = m[n][1] == -INFINITY ? 0.f : m[n][1];
      const float p0 = ex2(x[0] - ref0), p1 = ex2(x[1] - ref1);
      const float p2 = ex2(x[2] - ref0), p3 = ex2(x[3] - ref1);
      l[n][0] += p0 + p2;
      l[n][1] += p1 + p3;
      // The weights are rounded to bf16 for the product alone; l keeps them whole.
      pb[n][0] = transpose8x8(pack_bf16(p0, p1));
      pb[n][1] = transpose8x8(pack_bf16(p2, p3));
    }
#pragma unroll
    for (int h = 0; h < VH; ++h) {
      const uint32_t* x = reinterpret_cast<const uint32_t*>(&vf[0][h]);
      const uint32_t* y = reinterpret_cast<const uint32_t*>(&vf[1][h]);
      const uint32_t* z = reinterpret_cast<const uint32_t*>(&vf[2][h]);
      const uint32_t* w = reinterpret_cast<const uint32_t*>(&vf[3][h]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t a0 = __byte_perm(x[j], y[j], 0x5410), a1 = __byte_perm(x[j], y[j], 0x7632);
        const uint32_t a2 = __byte_perm(z[j], w[j], 0x5410), a3 = __byte_perm(z[j], w[j], 0x7632);
#pragma unroll
        for (int n = 0; n < NQ; ++n) mma16816(o[n][h][j], a0, a1, a2, a3, pb[n][0], pb[n][1]);
      }
    }
    if (next < k1) load_v(row_next);
  }

  // Whole sums of the rows' weights.
#pragma unroll
  for (int n = 0; n < NQ; ++n)
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int w = 4; w <= 16; w <<= 1) l[n][u] += __shfl_xor_sync(0xffffffffu, l[n][u], w);

  // The only part of its row also takes in the prefix's parts, dealt out to
  // the warps: lane (gq, t) holds d = 64h + 8 gq .. + 7 of rows 2t, 2t + 1.
  if (parts == 1) {
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const int r = 8 * n + 2 * t;
      for (int slot = warp; slot < p.np; slot += kWarps) {
        float pm[2], pl[2], v[2][VH][8];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          pm[u] = -INFINITY;
          pl[u] = 0.f;
          const int64_t at = (static_cast<int64_t>(g) * p.rows + row0 + r + u) * p.ns + slot;
          const bool ok = r + u < nrows;
          if (ok) {
            pm[u] = p.ml[at * 2];
            pl[u] = p.ml[at * 2 + 1];
          }
#pragma unroll
          for (int h = 0; h < VH; ++h)
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
              float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
              if (ok && gq + 8 * h < nchunks)
                f = *reinterpret_cast<const float4*>(p.acc + at * p.D + 64 * h + 8 * gq + e);
              v[u][h][e] = f.x, v[u][h][e + 1] = f.y, v[u][h][e + 2] = f.z, v[u][h][e + 3] = f.w;
            }
        }
        if (pm[0] > m[n][0] || pm[1] > m[n][1])
          rescale(n, fmaxf(m[n][0], pm[0]), fmaxf(m[n][1], pm[1]));
        const float f0 = pm[0] == -INFINITY ? 0.f : ex2(pm[0] - m[n][0]);
        const float f1 = pm[1] == -INFINITY ? 0.f : ex2(pm[1] - m[n][1]);
        l[n][0] += f0 * pl[0];
        l[n][1] += f1 * pl[1];
#pragma unroll
        for (int h = 0; h < VH; ++h)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            o[n][h][j][0] += f0 * v[0][h][2 * j];
            o[n][h][j][1] += f1 * v[1][h][2 * j];
            o[n][h][j][2] += f0 * v[0][h][2 * j + 1];
            o[n][h][j][3] += f1 * v[1][h][2 * j + 1];
          }
      }
    }
  }

  // The warps' states meet in shared memory.
#pragma unroll
  for (int n = 0; n < NQ; ++n)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int r = 8 * n + 2 * t + u;
      if (gq == 0) {
        s_m[warp][r] = m[n][u];
        s_l[warp][r] = l[n][u];
      }
#pragma unroll
      for (int h = 0; h < VH; ++h) {
        float* dst = &s_o[warp][r][64 * h + 8 * gq];
        *reinterpret_cast<float4*>(dst) =
            make_float4(o[n][h][0][u], o[n][h][0][u + 2], o[n][h][1][u], o[n][h][1][u + 2]);
        *reinterpret_cast<float4*>(dst + 4) =
            make_float4(o[n][h][2][u], o[n][h][2][u + 2], o[n][h][3][u], o[n][h][3][u + 2]);
      }
    }
  __syncthreads();
  for (int i = threadIdx.x; i < nrows * nchunks; i += kWarps * 32) {
    const int r = i / nchunks, d0 = (i % nchunks) * 8;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) M = fmaxf(M, s_m[w][r]);
    float L = 0.f, a[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) a[e] = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = s_m[w][r] == -INFINITY ? (s_l[w][r] == 0.f ? 0.f : 1.f) : ex2(s_m[w][r] - M);
      L = fmaf(f, s_l[w][r], L);
#pragma unroll
      for (int e = 0; e < 8; ++e) a[e] = fmaf(f, s_o[w][r][d0 + e], a[e]);
    }
    if (parts == 1) {
      const float inv = 1.0f / L;
#pragma unroll
      for (int e = 0; e < 8; ++e) a[e] *= inv;
      const int64_t at = b * p.os0 + (g * p.rep + chunk * R + r) * p.os1 + d0 * p.os2;
      if (op.out_vec) {
        *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.out) + at) =
            make_uint4(pack_bf16(a[0], a[1]), pack_bf16(a[2], a[3]), pack_bf16(a[4], a[5]),
                       pack_bf16(a[6], a[7]));
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) store_elem(p.out, at + e * p.os2, p.out_dtype, a[e]);
      }
    } else {
      const int64_t at = (static_cast<int64_t>(g) * p.rows + row0 + r) * p.ns + p.np + split;
      float4* dst = reinterpret_cast<float4*>(p.acc + at * p.D + d0);
      dst[0] = make_float4(a[0], a[1], a[2], a[3]);
      dst[1] = make_float4(a[4], a[5], a[6], a[7]);
      if (d0 == 0) {
        p.ml[at * 2] = M;
        p.ml[at * 2 + 1] = L;
      }
    }
  }
  if (parts == 1) return;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    const int64_t unit = (static_cast<int64_t>(b) * p.Hkv + g) * p.row_chunks + chunk;
    s_last = atomicAdd(&p.cnt[unit], 1) == parts - 1;
  }
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  for (int r = warp; r < nrows; r += kWarps) join_row(p, g, row0 + r, parts, lane, 32);
}

template <int DP, int NQ>
int launch(const OwnParams& op, cudaStream_t stream) {
  const SharedParams& p = op.s;
  const int64_t grid = static_cast<int64_t>(p.B) * p.own_splits * p.row_chunks * p.Hkv;
  if (grid > 0x7fffffffLL) return fail(B200_ERR_UNSUPPORTED, "shared prefix: grid too large");
  shared_own_mma_kernel<DP, NQ><<<static_cast<unsigned>(grid), kWarps * 32, 0, stream>>>(op);
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? B200_OK : cuda_fail(e, "shared prefix own-key launch");
}

bool vec16(const void* p, int64_t s0, int64_t s1, int64_t s2) {
  return s2 == 1 && reinterpret_cast<uintptr_t>(p) % 16 == 0 && s0 % 8 == 0 && s1 % 8 == 0;
}

}  // namespace

int shared_own_rows(int64_t rep) { return rep <= 8 ? 8 : 16; }

int launch_shared_own_mma(const SharedParams& p, cudaStream_t stream) {
  OwnParams op;
  op.s = p;
  op.q_vec = vec16(p.q, p.qs0, p.qs1, p.qs2);
  op.out_vec = p.out_dtype == B200_DTYPE_BF16 && vec16(p.out, p.os0, p.os1, p.os2);
  const bool wide = shared_own_rows(p.rep) == 16;
  if (p.D <= 64) return wide ? launch<64, 2>(op, stream) : launch<64, 1>(op, stream);
  return wide ? launch<128, 2>(op, stream) : launch<128, 1>(op, stream);
}

}  // namespace b200
