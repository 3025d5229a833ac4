// rope.cu -- per-head RMS norm and position rotation of q and k, with or
// without the append of k and v to the paged KV pool (CUDA cores, HBM-bound).
//
// For a head row x of D elements of token t at position n = positions[t]:
//   y = x * rsqrt(sum(x^2) / D + eps) * w            (rows with a weight)
//   (y_a, y_b) -> (y_a c_i - y_b s_i, y_a s_i + y_b c_i)   for i < R / 2
// where c_i, s_i come from the f32 table row n and (a, b) = (i, i + R/2), or
// (2i, 2i + 1) in the interleaved form.  All in f32, one rounding at the
// store.  Every element is read once and written once, so the floor is the
// bytes; what a small call costs is the launch and the chain position ->
// table row -> store.
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "host_util.h"
#include "kernels.h"

namespace b200 {
namespace {

struct RopeParams {
  const void* q;
  const void* k;
  const void* v;  // append only
  void* q_out;
  void* k_out;  // norm + rotation only
  void* k_pool;
  void* v_pool;
  int64_t qs0, qs1, qs2, ks0, ks1, ks2, vs0, vs1, vs2;
  int64_t qo0, qo1, qo2, ko0, ko1, ko2;
  const void* q_weight;
  const void* k_weight;
  const float* cos_sin;
  int64_t table_rows;
  const void* positions;
  int64_t pos_stride;
  const void* slots;
  int64_t slot_stride;
  int64_t pool_slots;  // P * S
  int64_t layer_row0;  // layer * P * S
  int32_t* status;
  int32_t Hq, Hkv, D, R;
  int32_t rows;  // head rows per token: Hq + Hkv (+ Hkv values)
  int32_t dtype, weight_dtype, pool_dtype;
  int32_t pos_i64, slots_i64, interleaved, append;
  float eps, inv_d;
};

__device__ __forceinline__ float2 fmul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
      "mul.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// One chunk (16, 8 or, of 16-bit types, 4 bytes) of the input type: N elements, as N / 2 pairs of floats.
template <typename T, int BYTES>
struct Chunk {
  static constexpr int N = BYTES / sizeof(T);
  using Raw = std::conditional_t<BYTES == 16, uint4, std::conditional_t<BYTES == 8, uint2, uint32_t>>;
  __device__ __forceinline__ static void unpack(const Raw& c, float2* f) {
    uint32_t w[BYTES / 4];
    if constexpr (BYTES == 4) w[0] = c;
    if constexpr (BYTES >= 8) w[0] = c.x, w[1] = c.y;
    if constexpr (BYTES == 16) w[2] = c.z, w[3] = c.w;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < N / 2; ++i)
        f[i] = make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
    } else {
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        if constexpr (std::is_same<T, __half>::value)
          f[i] = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        else
          f[i] = bf16x2_to_float2(w[i]);
      }
    }
  }
};

// P pairs of floats, 16 bytes at a time where P is even.
template <int P>
__device__ __forceinline__ void load_floats(const float* src, float2* f) {
  if constexpr (P == 1) {
    f[0] = __ldg(reinterpret_cast<const float2*>(src));
  } else {
#pragma unroll
    for (int i = 0; i < P; i += 2) {
      const float4 x = __ldg(reinterpret_cast<const float4*>(src + 2 * i));
      f[i] = make_float2(x.x, x.y);
      f[i + 1] = make_float2(x.z, x.w);
    }
  }
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float2 f) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(f.x, f.y);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

// Stores P (1, 2 or 4) pairs as T.
template <typename T, int P>
__device__ __forceinline__ void store_chunk(T* dst, const float2* f) {
  if constexpr (sizeof(T) == 4 && P == 1) {
    *reinterpret_cast<float2*>(dst) = f[0];
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < P; i += 2)
      *reinterpret_cast<float4*>(dst + 2 * i) = make_float4(f[i].x, f[i].y, f[i + 1].x, f[i + 1].y);
  } else if constexpr (P == 4) {
    *reinterpret_cast<uint4*>(dst) =
        make_uint4(pack2<T>(f[0]), pack2<T>(f[1]), pack2<T>(f[2]), pack2<T>(f[3]));
  } else if constexpr (P == 2) {
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(f[0]), pack2<T>(f[1]));
  } else {
    *reinterpret_cast<uint32_t*>(dst) = pack2<T>(f[0]);
  }
}

// The weights of one chunk (input type or f32).
template <typename In, int BYTES>
__device__ __forceinline__ void load_weight(const void* w, int weight_dtype, int e0, float2* f) {
  using C = Chunk<In, BYTES>;
  if (weight_dtype == B200_DTYPE_F32)
    load_floats<C::N / 2>(static_cast<const float*>(w) + e0, f);
  else
    C::unpack(__ldg(reinterpret_cast<const typename C::Raw*>(static_cast<const In*>(w) + e0)), f);
}

enum RowKind { kRowQ = 0, kRowK = 1, kRowV = 2 };

constexpr int kJobWarps = 4;  // warps per CTA


// Vector path.  A round is the head rows a warp takes side by side, a job up to
// U rounds of one kind (queries, keys, values) of a token; a warp per job,
// tokens' jobs end to end.  LPH lanes (a power of two)
// share a head row, lane j owning two chunks of 16 (8, 4) bytes: (j, j + R/2) of the
// rotated part in the split form, (2j, 2j + 1) otherwise, so that both elements
// of every pair are in one lane, and the pairs of lane j are i = j N .. j N + N
// - 1 in either form.  Norm weight and rotation are combined once per job into
//   a' = a A + o B,   b' = b C + o' D     (o, o' the chunks' partners)
// so that a row costs two packed products an element pair; all loads of a job
// are on their way before the first sum.  Each lane writes exactly the
// elements that it read, so q_out may be q.
// 8192 tokens of 32 + 8 heads of 128, bf16: 35 us, 4.9 TB/s (27 us at the copy
// rate), 32 + 32 heads with the append 67 us, 6.1 TB/s (64); with a row's kind,
// weights and addresses worked out row by row 57 and 108 us, bound by
// instructions.  U: 4 where the warps fill the GPU all the same (with 2: 38 and
// 78 us), else 2 (64 tokens: 2.8 us, with 4: 3.3 us).
// SHIFT: log2(LPH) where it is known (heads of 128), else -1.
template <typename In, typename PoolT, bool INTER, int SHIFT, int U, int BYTES>
__global__ void __launch_bounds__(kJobWarps * 32)
    rope_vec_kernel(const __grid_constant__ RopeParams p, const int shift_arg, const uint32_t jobs_q,
                    const uint32_t jobs_k, const uint32_t jobs, const uint32_t all_jobs, const int64_t t0) {
  using Ch = Chunk<In, BYTES>;
  using Raw = typename Ch::Raw;
  constexpr int N = Ch::N, P = N / 2;
  const int lph_shift = SHIFT >= 0 ? SHIFT : shift_arg;
  const int lane = threadIdx.x & 31;
  const uint32_t index = blockIdx.x * kJobWarps + (threadIdx.x >> 5);
  if (index >= all_jobs) return;
  const uint32_t token = index / jobs;  // of this launch
  const uint32_t job = index - token * jobs;
  const int64_t t = t0 + token;
  const int j = lane & ((1 << lph_shift) - 1);
  const int sub = lane >> lph_shift;     // row of a round
  const int rpw = 32 >> lph_shift;       // rows of a round
  const int pairs = p.D / (2 * N);       // lanes that own chunks
  const int turned = p.R / (2 * N);      // of which these are rotated
  const bool mine = j < pairs;
  const bool rot = j < turned;
  const bool split = rot && !INTER;
  const int ea = (split ? j : 2 * j) * N;               // first element of chunk a
  const int eb = (split ? j + turned : 2 * j + 1) * N;  // and of chunk b

  const int64_t pos = load_index(p.positions, t * p.pos_stride, p.pos_i64);
  const int64_t slot = p.append ? load_index(p.slots, t * p.slot_stride, p.slots_i64) : 0;
  const int kind = job < jobs_q ? kRowQ : job < jobs_q + jobs_k ? kRowK : kRowV;
  const int row0 = static_cast<int>(kind == kRowQ   ? job
                                    : kind == kRowK ? job - jobs_q
                                                    : job - jobs_q - jobs_k) * (U * rpw) + sub;
  const int rows = kind == kRowQ ? p.Hq : p.Hkv;
  const In* src = kind == kRowQ   ? static_cast<const In*>(p.q) + t * p.qs0
                  : kind == kRowK ? static_cast<const In*>(p.k) + t * p.ks0
                                  : static_cast<const In*>(p.v) + t * p.vs0;
  const int64_t step = kind == kRowQ ? p.qs1 : kind == kRowK ? p.ks1 : p.vs1;
  src += row0 * step;
  Raw ca[U], cb[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    ca[u] = cb[u] = Raw{};
    if (mine && row0 + u * rpw < rows) {
      ca[u] = *reinterpret_cast<const Raw*>(src + u * rpw * step + ea);
      cb[u] = *reinterpret_cast<const Raw*>(src + u * rpw * step + eb);
    }
  }
  const bool pos_ok = pos >= 0 && pos < p.table_rows;
  const bool slot_ok = !p.append || (slot >= 0 && slot < p.pool_slots);
  if (job == 0 && lane == 0 && !(pos_ok && slot_ok))
    report(p.status, (pos_ok ? 0 : B200_DEV_BAD_POSITION) | (slot_ok ? 0 : B200_DEV_BAD_SLOT));
  const bool to_pool = p.append && kind != kRowQ;
  In* out = nullptr;
  int64_t out_step = 0;
  if (!to_pool) {
    out = kind == kRowQ ? static_cast<In*>(p.q_out) + t * p.qo0 : static_cast<In*>(p.k_out) + t * p.ko0;
    out_step = kind == kRowQ ? p.qo1 : p.ko1;
    out += row0 * out_step;
  }
  if (!(pos_ok && (slot_ok || !to_pool))) {  // nothing for the pool, zeros for the rest
    float2 z[P];
#pragma unroll
    for (int i = 0; i < P; ++i) z[i] = make_float2(0.f, 0.f);
    for (int u = 0; u < U; ++u)
      if (!to_pool && mine && row0 + u * rpw < rows) {
        store_chunk<In, P>(out + u * rpw * out_step + ea, z);
        store_chunk<In, P>(out + u * rpw * out_step + eb, z);
      }
    return;
  }
  PoolT* pool = nullptr;
  if (to_pool)
    pool = static_cast<PoolT*>(kind == kRowK ? p.k_pool : p.v_pool) +
           ((p.layer_row0 + slot) * p.Hkv + row0) * p.D;

  if (kind == kRowV) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!mine || row0 + u * rpw >= rows) continue;
      PoolT* dst = pool + static_cast<int64_t>(u * rpw) * p.D;
      if constexpr (std::is_same<In, PoolT>::value) {  // values as they are
        *reinterpret_cast<Raw*>(dst + ea) = ca[u];
        *reinterpret_cast<Raw*>(dst + eb) = cb[u];
      } else {
        float2 f[P];
        Ch::unpack(ca[u], f);
        store_chunk<PoolT, P>(dst + ea, f);
        Ch::unpack(cb[u], f);
        store_chunk<PoolT, P>(dst + eb, f);
      }
    }
    return;
  }

  // A, C: the weights (times the cosines); B, D: the partners' sines.
  const void* weight = kind == kRowQ ? p.q_weight : p.k_weight;
  float2 A[P], B[P], C[P], D[P];
#pragma unroll
  for (int i = 0; i < P; ++i) A[i] = C[i] = make_float2(1.f, 1.f);
  if (weight != nullptr && mine) {
    load_weight<In, BYTES>(weight, p.weight_dtype, ea, A);
    load_weight<In, BYTES>(weight, p.weight_dtype, eb, C);
  }
  if (rot) {
    float2 c[P], s[P];
    const float* row = p.cos_sin + pos * p.R + j * N;
    load_floats<P>(row, c);
    load_floats<P>(row + p.R / 2, s);
    if constexpr (!INTER) {  // a' = a wa c - b wb s,  b' = b wb c + a wa s
#pragma unroll
      for (int i = 0; i < P; ++i) {
        B[i] = fmul2(C[i], make_float2(-s[i].x, -s[i].y));
        D[i] = fmul2(A[i], s[i]);
        A[i] = fmul2(A[i], c[i]);
        C[i] = fmul2(C[i], c[i]);
      }
    } else {  // (x, y)' = (x wx, y wy) c + (-y wy, x wx) s, a word of the chunk a pair
#pragma unroll
      for (int i = 0; i < P; ++i) {
        // Pair i of chunk a and pair P + i of the lane (chunk b).
        const float ca_ = i & 1 ? c[i / 2].y : c[i / 2].x, sa_ = i & 1 ? s[i / 2].y : s[i / 2].x;
        const float cb_ = (P + i) & 1 ? c[(P + i) / 2].y : c[(P + i) / 2].x;
        const float sb_ = (P + i) & 1 ? s[(P + i) / 2].y : s[(P + i) / 2].x;
        B[i] = make_float2(-A[i].y * sa_, A[i].x * sa_);
        D[i] = make_float2(-C[i].y * sb_, C[i].x * sb_);
        A[i] = make_float2(A[i].x * ca_, A[i].y * ca_);
        C[i] = make_float2(C[i].x * cb_, C[i].y * cb_);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < P; ++i) B[i] = D[i] = make_float2(0.f, 0.f);
  }

#pragma unroll
  for (int u = 0; u < U; ++u) {
    float2 a[P], b[P];
    Ch::unpack(ca[u], a);
    Ch::unpack(cb[u], b);
    if (weight != nullptr) {  // the same for the whole warp
      float2 ss = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < P; ++i) ss = ffma2(a[i], a[i], ffma2(b[i], b[i], ss));
      float sum = ss.x + ss.y;
#pragma unroll
      for (int o = 0; o < (SHIFT >= 0 ? SHIFT : 5); ++o)
        if (SHIFT >= 0 || o < lph_shift) sum += __shfl_xor_sync(0xffffffffu, sum, 1 << o);
      const float inv = rsqrtf(fmaf(sum, p.inv_d, p.eps));
      const float2 inv2 = make_float2(inv, inv);
#pragma unroll
      for (int i = 0; i < P; ++i) {
        a[i] = fmul2(a[i], inv2);
        b[i] = fmul2(b[i], inv2);
      }
    }
    if (!mine || row0 + u * rpw >= rows) continue;
    float2 x[P], y[P];
#pragma unroll
    for (int i = 0; i < P; ++i) {
      x[i] = fmul2(a[i], A[i]);
      y[i] = fmul2(b[i], C[i]);
      if (rot) {  // unrotated elements take nothing of a partner (0 * inf is NaN)
        x[i] = ffma2(INTER ? make_float2(a[i].y, a[i].x) : b[i], B[i], x[i]);
        y[i] = ffma2(INTER ? make_float2(b[i].y, b[i].x) : a[i], D[i], y[i]);
      }
    }
    if (to_pool) {
      PoolT* dst = pool + static_cast<int64_t>(u * rpw) * p.D;
      store_chunk<PoolT, P>(dst + ea, x);
      store_chunk<PoolT, P>(dst + eb, y);
    } else {
      In* dst = out + u * rpw * out_step;
      store_chunk<In, P>(dst + ea, x);
      store_chunk<In, P>(dst + eb, y);
    }
  }
}

// Any strides, alignment and sizes: a warp per head row, a lane per pair (or
// unrotated element), element loads.  As above every lane writes what it read.
__global__ void __launch_bounds__(256) rope_any_kernel(const RopeParams p) {
  const int64_t t = blockIdx.x;
  const int lane = threadIdx.x & 31;
  const int64_t pos = load_index(p.positions, t * p.pos_stride, p.pos_i64);
  const int64_t slot = p.append ? load_index(p.slots, t * p.slot_stride, p.slots_i64) : 0;
  const bool pos_ok = pos >= 0 && pos < p.table_rows;
  const bool slot_ok = !p.append || (slot >= 0 && slot < p.pool_slots);
  if (threadIdx.x == 0 && !(pos_ok && slot_ok))
    report(p.status, (pos_ok ? 0 : B200_DEV_BAD_POSITION) | (slot_ok ? 0 : B200_DEV_BAD_SLOT));
  const int half = p.R / 2;
  const int items = half + (p.D - p.R);  // pairs, then unrotated elements
  constexpr int kMax = 8;                // ceil(256 / 32)

  for (int r = threadIdx.x >> 5; r < p.rows; r += blockDim.x >> 5) {
    const int kind = r < p.Hq ? kRowQ : r < p.Hq + p.Hkv ? kRowK : kRowV;
    const int head = kind == kRowQ ? r : kind == kRowK ? r - p.Hq : r - p.Hq - p.Hkv;
    const void* src = kind == kRowQ ? p.q : kind == kRowK ? p.k : p.v;
    const int64_t base = kind == kRowQ   ? t * p.qs0 + head * p.qs1
                         : kind == kRowK ? t * p.ks0 + head * p.ks1
                                         : t * p.vs0 + head * p.vs1;
    const int64_t sd = kind == kRowQ ? p.qs2 : kind == kRowK ? p.ks2 : p.vs2;
    const void* w = kind == kRowQ ? p.q_weight : kind == kRowK ? p.k_weight : nullptr;
    float a[kMax], b[kMax];
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < kMax; ++i) {
      const int e = lane + 32 * i;
      a[i] = b[i] = 0.f;
      if (e < half) {
        a[i] = load_elem(src, base + (p.interleaved ? 2 * e : e) * sd, p.dtype);
        b[i] = load_elem(src, base + (p.interleaved ? 2 * e + 1 : e + half) * sd, p.dtype);
      } else if (e < items) {
        a[i] = load_elem(src, base + (p.R + e - half) * sd, p.dtype);
      }
      ss = fmaf(a[i], a[i], fmaf(b[i], b[i], ss));
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float inv = rsqrtf(fmaf(ss, p.inv_d, p.eps));
    void* dst;
    int64_t dbase, dd;
    int dst_dtype = p.dtype;
    if (kind == kRowQ || !p.append) {
      dst = kind == kRowQ ? p.q_out : p.k_out;
      dbase = kind == kRowQ ? t * p.qo0 + head * p.qo1 : t * p.ko0 + head * p.ko1;
      dd = kind == kRowQ ? p.qo2 : p.ko2;
    } else {
      if (!(pos_ok && slot_ok)) continue;
      dst = kind == kRowK ? p.k_pool : p.v_pool;
      dbase = ((p.layer_row0 + slot) * p.Hkv + head) * p.D;
      dd = 1;
      dst_dtype = p.pool_dtype;
    }
#pragma unroll
    for (int i = 0; i < kMax; ++i) {
      const int e = lane + 32 * i;
      if (e >= items) continue;
      const bool pair = e < half;
      const int d0 = !pair ? p.R + e - half : p.interleaved ? 2 * e : e;
      const int d1 = p.interleaved ? 2 * e + 1 : e + half;
      float x = a[i], y = b[i];
      if (w != nullptr) {
        x *= inv * load_elem(w, d0, p.weight_dtype);
        if (pair) y *= inv * load_elem(w, d1, p.weight_dtype);
      }
      if (pair && pos_ok && kind != kRowV) {
        const float c = __ldg(p.cos_sin + pos * p.R + e), s = __ldg(p.cos_sin + pos * p.R + half + e);
        const float x0 = x;
        x = x0 * c - y * s;
        y = x0 * s + y * c;
      }
      if (!pos_ok) x = y = 0.f;
      store_elem(dst, dbase + d0 * dd, dst_dtype, x);
      if (pair) store_elem(dst, dbase + d1 * dd, dst_dtype, y);
    }
  }
}

bool aligned(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// Access in chunks of `bytes` to every row of a [T, H, D] tensor.
bool rows_vec(const void* p, const int64_t* st, size_t es, int bytes) {
  return st[2] == 1 && aligned(p, bytes) && (st[0] * static_cast<int64_t>(es)) % bytes == 0 &&
         (st[1] * static_cast<int64_t>(es)) % bytes == 0;
}

template <typename In, typename PoolT, int U, int BYTES>
int launch_jobs(const RopeParams& p, int64_t tokens, cudaStream_t stream) {
  constexpr int N = Chunk<In, BYTES>::N;
  constexpr int kShift128 = BYTES < 16 ? -1 : N == 8 ? 3 : 4;
  const int shift = log2i(p.D / (2 * N));
  const int per_job = U * (32 >> shift);
  const uint32_t jobs_q = static_cast<uint32_t>(ceil_div(p.Hq, per_job));
  const uint32_t jobs_k = static_cast<uint32_t>(ceil_div(p.Hkv, per_job));
  const uint32_t jobs = jobs_q + jobs_k * (p.append ? 2 : 1);
  auto kern = shift == kShift128 ? (p.interleaved ? rope_vec_kernel<In, PoolT, true, kShift128, U, BYTES>
                                                  : rope_vec_kernel<In, PoolT, false, kShift128, U, BYTES>)
                                 : (p.interleaved ? rope_vec_kernel<In, PoolT, true, -1, U, BYTES>
                                                  : rope_vec_kernel<In, PoolT, false, -1, U, BYTES>);
  // Job numbers are 32-bit: very many tokens take several launches.
  const int64_t most = (int64_t(1) << 31) / jobs;
  for (int64_t t0 = 0; t0 < tokens; t0 += most) {
    const uint32_t all = static_cast<uint32_t>(std::min(most, tokens - t0) * jobs);
    kern<<<(all + kJobWarps - 1) / kJobWarps, kJobWarps * 32, 0, stream>>>(p, shift, jobs_q, jobs_k, jobs, all, t0);
  }
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? B200_OK : cuda_fail(e, "rotation launch");
}

template <typename In, typename PoolT>
int launch_vec(const RopeParams& p, int bytes, int64_t tokens, int num_sms, cudaStream_t stream) {
  const int shift = log2i(p.D / (2 * bytes / static_cast<int>(sizeof(In))));
  const int64_t rounds = tokens * (ceil_div(p.rows, 32 >> shift));
  // About 20 warps of four rounds to an SM.
  const bool four = rounds >= int64_t(4) * 20 * num_sms;
  if (bytes == 16)
    return four ? launch_jobs<In, PoolT, 4, 16>(p, tokens, stream) : launch_jobs<In, PoolT, 2, 16>(p, tokens, stream);
  if constexpr (sizeof(In) == 2)
    if (bytes == 4)
      return four ? launch_jobs<In, PoolT, 4, 4>(p, tokens, stream) : launch_jobs<In, PoolT, 2, 4>(p, tokens, stream);
  return four ? launch_jobs<In, PoolT, 4, 8>(p, tokens, stream) : launch_jobs<In, PoolT, 2, 8>(p, tokens, stream);
}

}  // namespace

int launch_qk_norm_rope(const b200_qk_norm_rope_args_t& a, const b200_rope_kv_append_args_t* append,
                        cudaStream_t stream) {
  DeviceInfo dev;
  int rc = current_device_info(&dev);
  if (rc != B200_OK) return rc;
  RopeParams p{};
  p.q = a.q;
  p.k = a.k;
  p.q_out = a.q_out;
  p.k_out = a.k_out;
  p.qs0 = a.q_stride[0], p.qs1 = a.q_stride[1], p.qs2 = a.q_stride[2];
  p.ks0 = a.k_stride[0], p.ks1 = a.k_stride[1], p.ks2 = a.k_stride[2];
  p.qo0 = a.q_out_stride[0], p.qo1 = a.q_out_stride[1], p.qo2 = a.q_out_stride[2];
  p.ko0 = a.k_out_stride[0], p.ko1 = a.k_out_stride[1], p.ko2 = a.k_out_stride[2];
  p.q_weight = a.q_weight;
  p.k_weight = a.k_weight;
  p.cos_sin = a.cos_sin;
  p.table_rows = a.table_rows;
  p.positions = a.positions;
  p.pos_stride = a.position_stride;
  p.status = a.status;
  p.Hq = static_cast<int32_t>(a.num_q_heads);
  p.Hkv = static_cast<int32_t>(a.num_kv_heads);
  p.D = static_cast<int32_t>(a.head_dim);
  p.R = static_cast<int32_t>(a.rotary_dim);
  p.rows = p.Hq + p.Hkv;
  p.dtype = a.dtype;
  p.weight_dtype = a.weight_dtype;
  p.pool_dtype = a.dtype;
  p.pos_i64 = a.position_dtype == B200_INDEX_I64;
  p.interleaved = a.interleaved != 0;
  p.eps = a.eps;
  p.inv_d = 1.0f / static_cast<float>(a.head_dim);
  if (append != nullptr) {
    p.append = 1;
    p.v = append->v;
    p.vs0 = append->v_stride[0], p.vs1 = append->v_stride[1], p.vs2 = append->v_stride[2];
    p.k_pool = append->pool.k;
    p.v_pool = append->pool.v;
    p.pool_dtype = append->pool.dtype;
    p.slots = append->slot_mapping;
    p.slot_stride = append->slot_stride;
    p.slots_i64 = append->slot_dtype == B200_INDEX_I64;
    p.pool_slots = append->pool.num_blocks * append->pool.block_size;
    p.layer_row0 = append->layer_idx * p.pool_slots;
    p.rows += p.Hkv;
  }
  // Chunks that every row's address and stride allow, in whole pairs: no lane
  // holds half of a rotated pair, and a warp at least a row.  (8192 tokens of 32 +
  // 8 heads of 80, 40 rotated, bf16: 34 us in chunks of 8 bytes, by elements 356;
  // 20 rotated: 57 us in chunks of 4, by elements 412.)
  const size_t es = dtype_size(a.dtype);
  auto fits = [&](int bytes) {
    const int n = bytes / static_cast<int>(es);
    if (!rows_vec(a.q, a.q_stride, es, bytes) || !rows_vec(a.k, a.k_stride, es, bytes) ||
        !rows_vec(a.q_out, a.q_out_stride, es, bytes) || !aligned(a.cos_sin, 16) ||
        !(append != nullptr ? rows_vec(append->v, append->v_stride, es, bytes)
                            : rows_vec(a.k_out, a.k_out_stride, es, bytes)))
      return false;
    if (p.D % (2 * n) != 0 || p.R % (2 * n) != 0 || p.D / (2 * n) > 32) return false;
    if (a.q_weight == nullptr && a.k_weight == nullptr) return true;
    return (a.weight_dtype == a.dtype || a.weight_dtype == B200_DTYPE_F32) &&
           (a.q_weight == nullptr || aligned(a.q_weight, 16)) &&
           (a.k_weight == nullptr || aligned(a.k_weight, 16));
  };
  const int vec = fits(16) ? 16 : fits(8) ? 8 : es == 2 && fits(4) ? 4 : 0;
  if (vec != 0) {
    const bool pool_f32 = p.pool_dtype == B200_DTYPE_F32;
    if (a.dtype == B200_DTYPE_F32) {
      if (pool_f32)
        rc = launch_vec<float, float>(p, vec, a.num_tokens, dev.num_sms, stream);
      else
        rc = launch_vec<float, __nv_bfloat16>(p, vec, a.num_tokens, dev.num_sms, stream);
    } else if (a.dtype == B200_DTYPE_BF16) {
      if (pool_f32)
        rc = launch_vec<__nv_bfloat16, float>(p, vec, a.num_tokens, dev.num_sms, stream);
      else
        rc = launch_vec<__nv_bfloat16, __nv_bfloat16>(p, vec, a.num_tokens, dev.num_sms, stream);
    } else {
      if (pool_f32)
        rc = launch_vec<__half, float>(p, vec, a.num_tokens, dev.num_sms, stream);
      else
        rc = launch_vec<__half, __nv_bfloat16>(p, vec, a.num_tokens, dev.num_sms, stream);
    }
    return rc;
  } else {
    const unsigned threads = static_cast<unsigned>(std::min(256, p.rows * 32));
    rope_any_kernel<<<static_cast<unsigned>(a.num_tokens), threads, 0, stream>>>(p);
  }
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "rotation launch");
  return B200_OK;
}

}  // namespace b200
