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

// Elem, Pack: one 16-byte chunk of the input type as floats and back.
template <typename T>
struct Chunk;
template <>
struct Chunk<float> {
  static constexpr int N = 4;
  __device__ __forceinline__ static void unpack(const uint4& c, float* f) { Elem<float>::unpack(c, f); }
};
template <>
struct Chunk<__nv_bfloat16> {
  static constexpr int N = 8;
  __device__ __forceinline__ static void unpack(const uint4& c, float* f) {
    Elem<__nv_bfloat16>::unpack(c, f);
  }
};
template <>
struct Chunk<__half> {
  static constexpr int N = 8;
  __device__ __forceinline__ static void unpack(const uint4& c, float* f) {
    const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = p.x;
      f[2 * i + 1] = p.y;
    }
  }
};

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (sizeof(T) == 2 && std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

// Stores N (4 or 8) consecutive floats as T, in 8- or 16-byte stores.
template <typename T, int N>
__device__ __forceinline__ void store_chunk(T* dst, const float* f) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < N; i += 4)
      *reinterpret_cast<float4*>(dst + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
  } else if constexpr (N == 8) {
    *reinterpret_cast<uint4*>(dst) = make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]),
                                                pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
  } else {
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]));
  }
}

// The weights of one chunk (input type or f32) as floats.
template <typename In>
__device__ __forceinline__ void load_weight(const void* w, int weight_dtype, int e0, float* f) {
  constexpr int N = Chunk<In>::N;
  if (weight_dtype == B200_DTYPE_F32) {
#pragma unroll
    for (int i = 0; i < N; i += 4)
      Elem<float>::unpack(__ldg(reinterpret_cast<const uint4*>(static_cast<const float*>(w) + e0 + i)),
                          f + i);
  } else {
    Chunk<In>::unpack(__ldg(reinterpret_cast<const uint4*>(static_cast<const In*>(w) + e0)), f);
  }
}

// Where a head row of a token lies: which tensor, which head.
enum RowKind { kRowQ = 0, kRowK = 1, kRowV = 2 };

// Vector path.  One CTA per token; LPH lanes (a power of two) share a head
// row, lane j owning two 16-byte chunks: (j, j + R/2) of the rotated part in
// the split form, (2j, 2j + 1) otherwise, so that both elements of every pair
// are in one lane, the pairs of lane j are i = j*N .. j*N + N - 1 in either
// form, and the table's values stay in registers over the token's rows.  Each
// lane writes exactly the elements it read, so q_out may be q.
// A thread loads the chunks of up to U rows before it stores the first.
template <typename In, typename PoolT, int U>
__global__ void __launch_bounds__(256) rope_vec_kernel(const RopeParams p, const int lph_shift) {
  constexpr int N = Chunk<In>::N;
  const int64_t t = blockIdx.x;
  const int lph = 1 << lph_shift;
  const int j = threadIdx.x & (lph - 1);
  const int group = threadIdx.x >> lph_shift;
  const int groups = blockDim.x >> lph_shift;
  const int pairs = p.D / (2 * N);   // lanes that own chunks
  const int turned = p.R / (2 * N);  // of which these are rotated
  const bool mine = j < pairs;
  const bool rot = j < turned;
  const bool split = rot && !p.interleaved;
  const int ea = (split ? j : 2 * j) * N;                   // first element of chunk a
  const int eb = (split ? j + turned : 2 * j + 1) * N;      // and of chunk b

  const int64_t pos = load_index(p.positions, t * p.pos_stride, p.pos_i64);
  const int64_t slot = p.append ? load_index(p.slots, t * p.slot_stride, p.slots_i64) : 0;
  const bool pos_ok = pos >= 0 && pos < p.table_rows;
  const bool slot_ok = !p.append || (slot >= 0 && slot < p.pool_slots);
  if (threadIdx.x == 0 && !(pos_ok && slot_ok))
    report(p.status, (pos_ok ? 0 : B200_DEV_BAD_POSITION) | (slot_ok ? 0 : B200_DEV_BAD_SLOT));

  float c[N], s[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    c[i] = 1.f;
    s[i] = 0.f;
  }
  if (rot && pos_ok) {
    const float* row = p.cos_sin + pos * p.R + j * N;
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      Elem<float>::unpack(__ldg(reinterpret_cast<const uint4*>(row + i)), c + i);
      Elem<float>::unpack(__ldg(reinterpret_cast<const uint4*>(row + p.R / 2 + i)), s + i);
    }
  }

  for (int r0 = group; r0 - group < p.rows; r0 += U * groups) {
    uint4 ca[U], cb[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = r0 + u * groups;
      ca[u] = cb[u] = make_uint4(0, 0, 0, 0);
      if (r < p.rows && mine) {
        const In* src;
        if (r < p.Hq)
          src = static_cast<const In*>(p.q) + t * p.qs0 + r * p.qs1;
        else if (r < p.Hq + p.Hkv)
          src = static_cast<const In*>(p.k) + t * p.ks0 + (r - p.Hq) * p.ks1;
        else
          src = static_cast<const In*>(p.v) + t * p.vs0 + (r - p.Hq - p.Hkv) * p.vs1;
        ca[u] = *reinterpret_cast<const uint4*>(src + ea);
        cb[u] = *reinterpret_cast<const uint4*>(src + eb);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      // Uniform over the row's lanes, not over the warp: every lane takes
      // part in the shuffles below.
      const int r = r0 + u * groups;
      const int kind = r < p.Hq ? kRowQ : r < p.Hq + p.Hkv ? kRowK : kRowV;
      float a[N], b[N];
      Chunk<In>::unpack(ca[u], a);
      Chunk<In>::unpack(cb[u], b);
      const void* w = kind == kRowQ ? p.q_weight : kind == kRowK ? p.k_weight : nullptr;
      if (p.q_weight != nullptr || p.k_weight != nullptr) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) ss = fmaf(a[i], a[i], fmaf(b[i], b[i], ss));
        for (int o = lph >> 1; o >= 1; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (w != nullptr && mine) {
          const float inv = rsqrtf(fmaf(ss, p.inv_d, p.eps));
          float wa[N], wb[N];
          load_weight<In>(w, p.weight_dtype, ea, wa);
          load_weight<In>(w, p.weight_dtype, eb, wb);
#pragma unroll
          for (int i = 0; i < N; ++i) {
            a[i] *= inv * wa[i];
            b[i] *= inv * wb[i];
          }
        }
      }
      if (r >= p.rows || !mine) continue;
      if (kind != kRowV && rot) {
        if (!p.interleaved) {
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const float x = a[i], y = b[i];
            a[i] = x * c[i] - y * s[i];
            b[i] = x * s[i] + y * c[i];
          }
        } else {
          // Pair i of the lane: elements 2i, 2i + 1 of its 2N consecutive ones.
#pragma unroll
          for (int i = 0; i < N; ++i) {
            float& x0 = 2 * i < N ? a[(2 * i) % N] : b[(2 * i) % N];
            float& y0 = 2 * i < N ? a[(2 * i + 1) % N] : b[(2 * i + 1) % N];
            const float x = x0, y = y0;
            x0 = x * c[i] - y * s[i];
            y0 = x * s[i] + y * c[i];
          }
        }
      }
      if (!pos_ok) {
#pragma unroll
        for (int i = 0; i < N; ++i) a[i] = b[i] = 0.f;
      }
      if (kind == kRowQ || !p.append) {
        In* dst = kind == kRowQ ? static_cast<In*>(p.q_out) + t * p.qo0 + r * p.qo1
                                : static_cast<In*>(p.k_out) + t * p.ko0 + (r - p.Hq) * p.ko1;
        store_chunk<In, N>(dst + ea, a);
        store_chunk<In, N>(dst + eb, b);
      } else if (pos_ok && slot_ok) {
        const int head = kind == kRowK ? r - p.Hq : r - p.Hq - p.Hkv;
        PoolT* dst = static_cast<PoolT*>(kind == kRowK ? p.k_pool : p.v_pool) +
                     ((p.layer_row0 + slot) * p.Hkv + head) * p.D;
        if (std::is_same<In, PoolT>::value && kind == kRowV) {  // values as they are
          *reinterpret_cast<uint4*>(dst + ea) = ca[u];
          *reinterpret_cast<uint4*>(dst + eb) = cb[u];
        } else {
          store_chunk<PoolT, N>(dst + ea, a);
          store_chunk<PoolT, N>(dst + eb, b);
        }
      }
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

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// 16-byte access to every row of a [T, H, D] tensor.
bool rows_vec(const void* p, const int64_t* st, size_t es) {
  return st[2] == 1 && aligned16(p) && (st[0] * static_cast<int64_t>(es)) % 16 == 0 &&
         (st[1] * static_cast<int64_t>(es)) % 16 == 0;
}

template <typename In, typename PoolT>
void launch_vec(const RopeParams& p, int64_t tokens, int num_sms, cudaStream_t stream) {
  constexpr int N = Chunk<In>::N;
  const int pairs = p.D / (2 * N);
  const int shift = log2i(pairs);
  const int lph = 1 << shift;
  // Up to 256 threads per token, the token's rows dealt out evenly.
  const int groups_max = 256 / lph;
  const int iters = static_cast<int>(ceil_div(p.rows, groups_max));
  const int groups = static_cast<int>(ceil_div(p.rows, iters));
  const unsigned threads = static_cast<unsigned>((groups * lph + 31) / 32 * 32);
  const unsigned grid = static_cast<unsigned>(tokens);
  if (iters == 1)
    rope_vec_kernel<In, PoolT, 1><<<grid, threads, 0, stream>>>(p, shift);
  else if (iters == 2)
    rope_vec_kernel<In, PoolT, 2><<<grid, threads, 0, stream>>>(p, shift);
  else
    rope_vec_kernel<In, PoolT, 3><<<grid, threads, 0, stream>>>(p, shift);
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
  const size_t es = dtype_size(a.dtype);
  bool vec = rows_vec(a.q, a.q_stride, es) && rows_vec(a.k, a.k_stride, es) &&
             rows_vec(a.q_out, a.q_out_stride, es) && aligned16(a.cos_sin);
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
    vec = vec && rows_vec(append->v, append->v_stride, es);
  } else {
    vec = vec && rows_vec(a.k_out, a.k_out_stride, es);
  }
  // Whole chunk pairs: no lane holds half of a rotated pair.
  const int n = static_cast<int>(16 / es);
  vec = vec && p.D % (2 * n) == 0 && p.R % (2 * n) == 0;
  if (a.q_weight != nullptr || a.k_weight != nullptr)
    vec = vec && (a.weight_dtype == a.dtype || a.weight_dtype == B200_DTYPE_F32) &&
          (a.q_weight == nullptr || aligned16(a.q_weight)) &&
          (a.k_weight == nullptr || aligned16(a.k_weight));
  if (vec) {
    const bool pool_f32 = p.pool_dtype == B200_DTYPE_F32;
    if (a.dtype == B200_DTYPE_F32) {
      if (pool_f32)
        launch_vec<float, float>(p, a.num_tokens, dev.num_sms, stream);
      else
        launch_vec<float, __nv_bfloat16>(p, a.num_tokens, dev.num_sms, stream);
    } else if (a.dtype == B200_DTYPE_BF16) {
      if (pool_f32)
        launch_vec<__nv_bfloat16, float>(p, a.num_tokens, dev.num_sms, stream);
      else
        launch_vec<__nv_bfloat16, __nv_bfloat16>(p, a.num_tokens, dev.num_sms, stream);
    } else {
      if (pool_f32)
        launch_vec<__half, float>(p, a.num_tokens, dev.num_sms, stream);
      else
        launch_vec<__half, __nv_bfloat16>(p, a.num_tokens, dev.num_sms, stream);
    }
  } else {
    const unsigned threads = static_cast<unsigned>(std::min(256, p.rows * 32));
    rope_any_kernel<<<static_cast<unsigned>(a.num_tokens), threads, 0, stream>>>(p);
  }
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "rotation launch");
  return B200_OK;
}

}  // namespace b200
