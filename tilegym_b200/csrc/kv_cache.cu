// Rotary positions, and the paged key / value cache in e4m3: writing it (with the rotation in front) and reading it back.
//
// The cache is laid out for the attention that reads it: a page holds 128 tokens of a head, keys as [token][dim] and values
// as [dim][token], so that both are K-major operands of the tensor core's 8-bit products as they lie in memory, and every
// (page, head) block has one scale for its keys and one for its values.  Scales are powers of two: dividing by one is
// exact, a value of the cache is exact in bf16, and a block whose scale has to grow, because a later token is larger than
// all before it, is moved to the new scale by changing exponents (only what falls below the format's normal range rounds
// again).  e4m3 keeps its 2^-4 relative rounding wherever a value sits in its range, so a power of two costs at most the
// lowest of 18 octaves.
#include <cstdio>

#include "tg_decoder_common.cuh"

namespace tg {
namespace {

struct RopeParams {
  const double* inv_freq;  // rotary / 2, radians per position
  int32_t rotary;          // elements of a head that are rotated (a multiple of 16)
  int32_t interleaved;
  float magnitude;
};

// ------------------------------------------------------------------------------------------ apply_rope
struct RopeHeads {
  const void* in;
  void* out;
  int64_t in_tok, in_head, out_tok, out_head;  // pitches in elements
  int32_t heads;
};
struct ApplyRopeParams {
  RopeHeads part[2];  // q and k
  RopeParams rope;
  const void* positions;
  int32_t positions64;
  int32_t units;    // dim / 16
  int32_t skip;     // in place: the units behind the rotated ones need no copy
};

constexpr int kMaxPairs = 256;

// One token's heads: cos and sin of its angles once in shared memory, then 16 elements at a time.
template <typename T>
__device__ __forceinline__ void rotate_heads(const RopeHeads& h, int64_t tok, int units_per_head, int units_done, int first, int stride,
                                             const RopeParams& r, const float2* cs) {
  const T* in = static_cast<const T*>(h.in) + tok * h.in_tok;
  T* out = static_cast<T*>(h.out) + tok * h.out_tok;
  for (int u = first; u < h.heads * units_done; u += stride) {
    const int head = u / units_done, w = u - head * units_done;
    int oa, ob, pair;
    unit_offsets(w, r.rotary, r.interleaved != 0, oa, ob, pair);
    uint4 a = *reinterpret_cast<const uint4*>(in + head * h.in_head + oa);
    uint4 b = *reinterpret_cast<const uint4*>(in + head * h.in_head + ob);
    if (pair >= 0) {
      float2 c[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) c[i] = cs[pair + i];
      rotate_unit<T>(a, b, c, r.interleaved != 0);
    }
    *reinterpret_cast<uint4*>(out + head * h.out_head + oa) = a;
    *reinterpret_cast<uint4*>(out + head * h.out_head + ob) = b;
  }
}

template <typename T>
__global__ void __launch_bounds__(256) tg_apply_rope_kernel(const ApplyRopeParams p) {
  __shared__ float2 cs[kMaxPairs];
  const int64_t tok = blockIdx.x;
  griddep_wait();
  griddep_launch_dependents();
  const int64_t pos = p.positions64 ? static_cast<const int64_t*>(p.positions)[tok] : static_cast<const int32_t*>(p.positions)[tok];
  for (int i = threadIdx.x; i < p.rope.rotary / 2; i += blockDim.x)
    cs[i] = cos_sin_at(turn_fraction(p.rope.inv_freq[i]), pos, p.rope.magnitude);
  __syncthreads();
  const int done = p.skip ? p.rope.rotary / 16 : p.units;
  rotate_heads<T>(p.part[0], tok, p.units, done, threadIdx.x, blockDim.x, p.rope, cs);
  rotate_heads<T>(p.part[1], tok, p.units, done, threadIdx.x, blockDim.x, p.rope, cs);
}

// ------------------------------------------------------------------------------------------ kv_cache_write
struct WriteParams {
  CacheView c;
  const void* x[2];  // new keys, new values [tokens, heads, dim]
  int64_t tok_pitch[2], head_pitch[2];
  RopeParams rope;  // inv_freq null: keys are written as they come
  RopeHeads q;      // queries rotated beside the keys; heads 0: none
  int32_t tokens, tiles;
};

constexpr int kWriteThreads = 128;
constexpr int kTransposePitch = 144;  // bytes of a value row in shared memory

__device__ __forceinline__ float block_max_128(float v, float* scratch) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  return fmaxf(fmaxf(scratch[0], scratch[1]), fmaxf(scratch[2], scratch[3]));
}

__device__ __forceinline__ float finite_abs(float v) {
  const float a = fabsf(v);
  return a <= 3.4028234e38f ? a : 0.f;
}

// e4m3 bytes times a power of two, rounded back to e4m3.
__device__ __forceinline__ uint32_t requantise4(uint32_t w, float f) {
  const __half2_raw lo = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w & 0xffffu), __NV_E4M3);
  const __half2_raw hi = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w >> 16), __NV_E4M3);
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo)), b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  return q8_cast2<kQ8E4M3>(a.x * f, a.y * f, 0.f, 0.f) | (q8_cast2<kQ8E4M3>(b.x * f, b.y * f, 0.f, 0.f) << 16);
}

// The bytes of w that lie below `keep` of its four are replaced by those of m.
__device__ __forceinline__ uint32_t merge_low(uint32_t w, uint32_t m, int keep) {
  if (keep >= 4) return m;
  if (keep <= 0) return w;
  const uint32_t mask = (1u << (8 * keep)) - 1u;
  return (w & ~mask) | (m & mask);
}

// A block owns one (page of a sequence, head) of the keys or of the values, so nobody else touches that block's scale or
// bytes.  The new values stay in registers between the maximum and the rounding (at most 8 units of 16 elements per
// thread); values go through shared memory on their way to [dim][token].
template <typename T, int DIM>
__device__ __forceinline__ void write_block(const WriteParams& p, int tile, int head, bool is_v, float2* table, uint8_t* bytes, float* red) {
  constexpr int kUnits = DIM / 16;                            // units of 16 elements per token
  constexpr int kPer = kPage * kUnits / kWriteThreads;        // units per thread when a whole page is new
  int first;
  const int b = find_sequence(p.c.cu, p.c.seqs, tile, kPage, 2, first);
  int lo, hi;
  new_rows(p.c.cu, b, p.tokens, lo, hi);
  const int len = p.c.seq_lens[b], start = len - (hi - lo);  // positions start .. len - 1 are new
  if (hi <= lo || len <= 0 || tile < first) return;
  const int page = max(start, 0) / kPage + (tile - first);
  if (page * kPage >= len || page >= p.c.max_pages) return;
  const int phys = p.c.table[b * p.c.table_pitch + page];
  if (phys < 0 || phys >= p.c.pages) return;
  const int t0 = max(start - page * kPage, 0), t1 = min(len - page * kPage, kPage);  // tokens of the page that are new
  const int64_t block = static_cast<int64_t>(phys) * p.c.heads + head;
  const int64_t row0 = static_cast<int64_t>(lo) + page * kPage - start;  // batch row of the page's token 0
  const T* x = static_cast<const T*>(p.x[is_v]) + head * p.head_pitch[is_v];
  const int count = (t1 - t0) * kUnits;
  const bool rope = !is_v && p.rope.inv_freq != nullptr;
  const bool inter = p.rope.interleaved != 0;
  const int rotary = rope ? p.rope.rotary : 0;

  uint4 va[kPer], vb[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int u = i * kWriteThreads + threadIdx.x;
    if (u < count) {
      const int t = t0 + u / kUnits;
      int oa, ob, pair;
      unit_offsets(u % kUnits, rotary, inter, oa, ob, pair);
      const T* src = x + (row0 + t) * p.tok_pitch[is_v];
      va[i] = *reinterpret_cast<const uint4*>(src + oa);
      vb[i] = *reinterpret_cast<const uint4*>(src + ob);
    } else {
      va[i] = vb[i] = make_uint4(0, 0, 0, 0);
    }
  }
  if (rope) {
    uint64_t* fraction = reinterpret_cast<uint64_t*>(table);
    for (int i = threadIdx.x; i < rotary / 2; i += kWriteThreads) fraction[i] = turn_fraction(p.rope.inv_freq[i]);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int u = i * kWriteThreads + threadIdx.x;
      const int w = u % kUnits;
      if (u < count && w * 16 < rotary) {
        const int pos = page * kPage + t0 + u / kUnits;
        float2 cs[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) cs[j] = cos_sin_at(fraction[w * 8 + j], pos, p.rope.magnitude);
        rotate_unit<T>(va[i], vb[i], cs, inter);
      }
    }
  }
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const uint32_t w[8] = {va[i].x, va[i].y, va[i].z, va[i].w, vb[i].x, vb[i].y, vb[i].z, vb[i].w};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float2 f = unpack_pair<T>(w[j]);
      amax = fmaxf(amax, fmaxf(finite_abs(f.x), finite_abs(f.y)));
    }
  }
  amax = block_max_128(amax, red);
  float s = cache_scale(amax);
  float* scale = (is_v ? p.c.vs : p.c.ks) + block;
  uint8_t* dst = (is_v ? p.c.v : p.c.k) + block * (kPage * DIM);
  if (t0 > 0) {
    const float old = *scale;
    if (old >= s) {
      s = old;
    } else {
      // earlier tokens of the page move to the larger scale
      const float f = old * pow2_reciprocal(s);
      if (is_v) {
        for (int i = threadIdx.x; i < DIM * (kPage / 16); i += kWriteThreads) {
          const int t = (i % (kPage / 16)) * 16;
          if (t >= t0) continue;
          uint4* at = reinterpret_cast<uint4*>(dst + (i / (kPage / 16)) * kPage + t);
          uint4 w = *at;
          w.x = merge_low(w.x, requantise4(w.x, f), t0 - t);
          w.y = merge_low(w.y, requantise4(w.y, f), t0 - t - 4);
          w.z = merge_low(w.z, requantise4(w.z, f), t0 - t - 8);
          w.w = merge_low(w.w, requantise4(w.w, f), t0 - t - 12);
          *at = w;
        }
      } else {
        for (int i = threadIdx.x; i < t0 * (DIM / 16); i += kWriteThreads) {
          uint4* at = reinterpret_cast<uint4*>(dst) + i;
          const uint4 w = *at;
          *at = make_uint4(requantise4(w.x, f), requantise4(w.y, f), requantise4(w.z, f), requantise4(w.w, f));
        }
      }
    }
    __syncthreads();  // the scale is read by all before it is written, old bytes are moved before new ones arrive
  }
  if (threadIdx.x == 0) *scale = s;
  const float r = pow2_reciprocal(s);
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int u = i * kWriteThreads + threadIdx.x;
    if (u >= count) continue;
    const int t = t0 + u / kUnits;
    int oa, ob, pair;
    unit_offsets(u % kUnits, rotary, inter, oa, ob, pair);
    const uint32_t w[8] = {va[i].x, va[i].y, va[i].z, va[i].w, vb[i].x, vb[i].y, vb[i].z, vb[i].w};
    uint32_t q[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f0 = unpack_pair<T>(w[2 * j]), f1 = unpack_pair<T>(w[2 * j + 1]);
      q[j] = q8_cast2<kQ8E4M3>(f0.x * r, f0.y * r, 0.f, 0.f) | (q8_cast2<kQ8E4M3>(f1.x * r, f1.y * r, 0.f, 0.f) << 16);
    }
    if (is_v) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        bytes[(oa + j) * kTransposePitch + t] = static_cast<uint8_t>(q[j >> 2] >> (8 * (j & 3)));
        bytes[(ob + j) * kTransposePitch + t] = static_cast<uint8_t>(q[2 + (j >> 2)] >> (8 * (j & 3)));
      }
    } else {
      *reinterpret_cast<uint2*>(dst + t * DIM + oa) = make_uint2(q[0], q[1]);
      *reinterpret_cast<uint2*>(dst + t * DIM + ob) = make_uint2(q[2], q[3]);
    }
  }
  if (is_v) {
    __syncthreads();
    for (int i = threadIdx.x; i < DIM * (kPage / 16); i += kWriteThreads) {
      const int d = i / (kPage / 16), t = (i % (kPage / 16)) * 16;
      const uint8_t* src = bytes + d * kTransposePitch + t;
      uint8_t* at = dst + d * kPage + t;
      if (t >= t0 && t + 16 <= t1) {
        *reinterpret_cast<uint4*>(at) = *reinterpret_cast<const uint4*>(src);
      } else {
        for (int j = max(t0 - t, 0); j < min(t1 - t, 16); ++j) at[j] = src[j];
      }
    }
  }
}

template <typename T, int DIM>
__global__ void __launch_bounds__(kWriteThreads) tg_kv_cache_write_kernel(const WriteParams p) {
  __shared__ __align__(16) uint8_t bytes[DIM * kTransposePitch];
  __shared__ float2 table[kMaxPairs];
  __shared__ float red[4];
  griddep_wait();
  griddep_launch_dependents();
  const int blocks = p.tiles * p.c.heads * 2;
  int id = blockIdx.x;
  if (id < blocks) {
    const int head = id % p.c.heads;
    id /= p.c.heads;
    write_block<T, DIM>(p, id >> 1, head, id & 1, table, bytes, red);
    return;
  }
  // the queries of one token
  const int tok = id - blocks;
  int first;
  // rows of the batch belong to the last sequence that starts at or before them
  const int b = find_sequence(p.c.cu, p.c.seqs, tok, 1, 0, first);
  int lo, hi;
  new_rows(p.c.cu, b, p.tokens, lo, hi);
  if (tok < lo || tok >= hi) return;  // rows behind the last sequence
  const int64_t pos = static_cast<int64_t>(p.c.seq_lens[b]) - hi + tok;
  for (int i = threadIdx.x; i < p.rope.rotary / 2; i += kWriteThreads)
    table[i] = cos_sin_at(turn_fraction(p.rope.inv_freq[i]), pos, p.rope.magnitude);
  __syncthreads();
  rotate_heads<T>(p.q, tok, DIM / 16, DIM / 16, threadIdx.x, kWriteThreads, p.rope, table);
}

// ------------------------------------------------------------------------------------------ kv_cache_read
struct ReadParams {
  CacheView c;
  void* out[2];
  int32_t max_len;
};

__device__ __forceinline__ float2 e4m3_pair(uint32_t two) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(two & 0xffffu), __NV_E4M3);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// A block turns one (page of a sequence, head) back into 16 bits; rows behind the sequence's length get zeros.
template <typename T, int DIM>
__global__ void __launch_bounds__(256) tg_kv_cache_read_kernel(const ReadParams p) {
  __shared__ __align__(16) uint8_t bytes[DIM * kTransposePitch];
  griddep_wait();
  griddep_launch_dependents();
  const int page = blockIdx.x, head = blockIdx.y >> 1, b = blockIdx.z;
  const bool is_v = blockIdx.y & 1;
  const int rows = min(p.max_len - page * kPage, kPage);
  const int len = p.c.seq_lens[b];
  int live = page < p.c.max_pages ? min(max(len - page * kPage, 0), rows) : 0;
  const int phys = live > 0 ? p.c.table[b * p.c.table_pitch + page] : 0;
  if (phys < 0 || phys >= p.c.pages) live = 0;
  const int64_t block = static_cast<int64_t>(phys) * p.c.heads + head;
  const uint8_t* src = (is_v ? p.c.v : p.c.k) + block * (kPage * DIM);
  const float s = live > 0 ? (is_v ? p.c.vs : p.c.ks)[block] : 0.f;
  T* out = static_cast<T*>(p.out[is_v]) +
           ((static_cast<int64_t>(b) * p.max_len + static_cast<int64_t>(page) * kPage) * p.c.heads + head) * DIM;
  const int64_t pitch = static_cast<int64_t>(p.c.heads) * DIM;
  if (is_v && live > 0) {
    for (int i = threadIdx.x; i < DIM * (kPage / 16); i += blockDim.x)
      *reinterpret_cast<uint4*>(bytes + (i / (kPage / 16)) * kTransposePitch + (i % (kPage / 16)) * 16) = reinterpret_cast<const uint4*>(src)[i];
    __syncthreads();
  }
  // 8 elements of a row per step
  for (int i = threadIdx.x; i < rows * (DIM / 8); i += blockDim.x) {
    const int t = i / (DIM / 8), d = (i % (DIM / 8)) * 8;
    uint4 o = make_uint4(0, 0, 0, 0);
    if (t < live) {
      uint32_t w[2];
      if (is_v) {
        w[0] = w[1] = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j >> 2] |= static_cast<uint32_t>(bytes[(d + j) * kTransposePitch + t]) << (8 * (j & 3));
      } else {
        const uint2 v = *reinterpret_cast<const uint2*>(src + t * DIM + d);
        w[0] = v.x;
        w[1] = v.y;
      }
      uint32_t r[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = e4m3_pair(w[j >> 1] >> (16 * (j & 1)));
        r[j] = pack_pair<T>(f.x * s, f.y * s);
      }
      o = make_uint4(r[0], r[1], r[2], r[3]);
    }
    __stcs(reinterpret_cast<uint4*>(out + t * pitch + d), o);
  }
}

int32_t launch_status(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return TG_OK;
  char msg[160];
  snprintf(msg, sizeof(msg), "%s launch failed: %s", what, cudaGetErrorString(e));
  return api_fail(TG_ERR_LAUNCH, msg);
}

int32_t check_rope(RopeParams* r, const TgTensorDesc* inv_freq, int64_t dim, int32_t interleaved, float magnitude) {
  if (inv_freq->ndim != 1 || inv_freq->dtype != TG_F64) return api_fail(TG_ERR_DTYPE, "inv_freq must be a float64 vector");
  const int64_t pairs = inv_freq->shape[0];
  if (pairs < 8 || pairs % 8 != 0 || 2 * pairs > dim)
    return api_fail(TG_ERR_ARGS, "inv_freq holds one value per rotated pair: a multiple of 8, at most head_dim / 2");
  if (inv_freq->strides[0] != 1) return api_fail(TG_ERR_ARGS, "inv_freq must be contiguous");
  if (inv_freq->ptr == 0) return api_fail(TG_ERR_NULL, "inv_freq pointer is null");
  if (inv_freq->ptr & 7u) return api_fail(TG_ERR_ALIGN, "inv_freq must be 8-byte aligned");
  r->inv_freq = reinterpret_cast<const double*>(inv_freq->ptr);
  r->rotary = static_cast<int32_t>(2 * pairs);
  r->interleaved = interleaved;
  r->magnitude = magnitude;
  return TG_OK;
}

RopeHeads heads_of(const TgTensorDesc* in, const TgTensorDesc* out) {
  return RopeHeads{reinterpret_cast<const void*>(in->ptr), reinterpret_cast<void*>(out->ptr), in->strides[0], in->strides[1],
                   out->strides[0], out->strides[1], static_cast<int32_t>(in->shape[1])};
}

int32_t select_device(int32_t device_id, int* num_sms) {
  int32_t* status = nullptr;
  return api_init_device(device_id, num_sms, &status);
}

}  // namespace
}  // namespace tg

using namespace tg;

extern "C" TG_API int32_t tg_apply_rope(const TgTensorDesc* Qo, const TgTensorDesc* Ko, const TgTensorDesc* Q, const TgTensorDesc* K,
                                        const TgTensorDesc* positions, const TgTensorDesc* inv_freq, int32_t interleaved, float magnitude,
                                        int32_t device_id, uint64_t stream) {
  if (Q == nullptr || positions == nullptr || inv_freq == nullptr) return api_fail(TG_ERR_NULL, "a descriptor is null");
  if (!is_16bit(Q->dtype)) return api_fail(TG_ERR_DTYPE, "q must be bf16 or f16");
  if (Q->ndim != 3) return api_fail(TG_ERR_ARGS, "q must be [tokens, heads, head_dim]");
  const int64_t T = Q->shape[0], D = Q->shape[2];
  if (T < 0 || T > 0x7fffffff) return api_fail(TG_ERR_ARGS, "too many tokens");
  if (D < 16 || D % 16 != 0 || D > 2 * kMaxPairs) return api_fail(TG_ERR_ARGS, "head_dim must be a multiple of 16 up to 512");
  if (Q->shape[1] < 1 || Q->shape[1] > 65536) return api_fail(TG_ERR_ARGS, "q needs 1 to 65536 heads");
  ApplyRopeParams p = {};
  int32_t rc;
  if ((rc = check_heads(Q, "q: rows of a head dense, pitches and pointer 16-byte aligned", T, Q->shape[1], D, Q->dtype)) != TG_OK) return rc;
  if ((rc = check_heads(Qo, "q output: shape and type of q, 16-byte aligned", T, Q->shape[1], D, Q->dtype)) != TG_OK) return rc;
  p.part[0] = heads_of(Q, Qo);
  if (K != nullptr) {
    if (K->ndim != 3 || K->shape[1] < 1 || K->shape[1] > 65536) return api_fail(TG_ERR_ARGS, "k must be [tokens, heads, head_dim]");
    if ((rc = check_heads(K, "k: tokens, head_dim and type of q, 16-byte aligned", T, K->shape[1], D, Q->dtype)) != TG_OK) return rc;
    if ((rc = check_heads(Ko, "k output: shape and type of k, 16-byte aligned", T, K->shape[1], D, Q->dtype)) != TG_OK) return rc;
    p.part[1] = heads_of(K, Ko);
  }
  if (positions->dtype != TG_I32 && positions->dtype != TG_I64) return api_fail(TG_ERR_DTYPE, "positions must be int32 or int64");
  const int64_t shape[1] = {T};
  if ((rc = check_dense_nd(positions, "positions: [tokens], contiguous", positions->dtype, 1, shape, positions->dtype == TG_I64 ? 8 : 4)) != TG_OK) return rc;
  if ((rc = check_rope(&p.rope, inv_freq, D, interleaved, magnitude)) != TG_OK) return rc;
  if (T == 0) return TG_OK;
  ScopedDevice guard(device_id);
  if (guard.err != cudaSuccess) {
    cudaGetLastError();
    return api_fail(TG_ERR_DEVICE, "cannot select the CUDA device");
  }
  int num_sms = 0;
  if ((rc = select_device(device_id, &num_sms)) != TG_OK) return rc;
  p.positions = reinterpret_cast<const void*>(positions->ptr);
  p.positions64 = positions->dtype == TG_I64;
  p.units = static_cast<int32_t>(D / 16);
  p.skip = p.part[0].in == p.part[0].out && p.part[1].in == p.part[1].out;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(T)), block(256);
  return launch_status(Q->dtype == TG_BF16 ? launch_pdl(tg_apply_rope_kernel<__nv_bfloat16>, grid, block, 0, st, p)
                                           : launch_pdl(tg_apply_rope_kernel<__half>, grid, block, 0, st, p),
                       "apply_rope");
}

extern "C" TG_API int32_t tg_kv_cache_write(const TgTensorDesc* Kc, const TgTensorDesc* Vc, const TgTensorDesc* Ks, const TgTensorDesc* Vs,
                                            const TgTensorDesc* K, const TgTensorDesc* V, const TgTensorDesc* block_table,
                                            const TgTensorDesc* seq_lens, const TgTensorDesc* cu_seqlens, const TgTensorDesc* Qo,
                                            const TgTensorDesc* Q, const TgTensorDesc* inv_freq, int32_t interleaved, float magnitude,
                                            int32_t device_id, uint64_t stream) {
  WriteParams p = {};
  int32_t rc;
  if ((rc = check_cache(&p.c, Kc, Vc, Ks, Vs, block_table, seq_lens, cu_seqlens)) != TG_OK) return rc;
  if (K == nullptr) return api_fail(TG_ERR_NULL, "k descriptor is null");
  if (!is_16bit(K->dtype)) return api_fail(TG_ERR_DTYPE, "k must be bf16 or f16");
  if (K->ndim != 3) return api_fail(TG_ERR_ARGS, "k must be [tokens, heads, head_dim]");
  const int64_t T = K->shape[0], D = p.c.dim;
  if (T > (1 << 28)) return api_fail(TG_ERR_ARGS, "too many tokens");
  if (cu_seqlens == nullptr && T != p.c.seqs) return api_fail(TG_ERR_ARGS, "without cu_seqlens there is one new token per sequence");
  if ((rc = check_heads(K, "k: [tokens, heads of the cache, head_dim], 16-byte aligned", T, p.c.heads, D, K->dtype)) != TG_OK) return rc;
  if ((rc = check_heads(V, "v: shape and type of k, 16-byte aligned", T, p.c.heads, D, K->dtype)) != TG_OK) return rc;
  if (inv_freq != nullptr && (rc = check_rope(&p.rope, inv_freq, D, interleaved, magnitude)) != TG_OK) return rc;
  if (Q != nullptr) {
    if (inv_freq == nullptr) return api_fail(TG_ERR_NULL, "queries are taken to be rotated: they need inv_freq");
    if (Q->ndim != 3 || Q->shape[1] < 1 || Q->shape[1] > 65536) return api_fail(TG_ERR_ARGS, "q must be [tokens, heads, head_dim]");
    if ((rc = check_heads(Q, "q: tokens, head_dim and type of k, 16-byte aligned", T, Q->shape[1], D, K->dtype)) != TG_OK) return rc;
    if ((rc = check_heads(Qo, "q output: shape and type of q, 16-byte aligned", T, Q->shape[1], D, K->dtype)) != TG_OK) return rc;
    p.q = heads_of(Q, Qo);
  }
  if (T == 0 || p.c.seqs == 0) return TG_OK;
  const int64_t tiles = T / kPage + 2 * static_cast<int64_t>(p.c.seqs);
  const int64_t blocks = tiles * p.c.heads * 2 + (Q ? T : 0);
  if (blocks > 0x7fffffff) return api_fail(TG_ERR_ARGS, "too many tokens and heads for one call");
  ScopedDevice guard(device_id);
  if (guard.err != cudaSuccess) {
    cudaGetLastError();
    return api_fail(TG_ERR_DEVICE, "cannot select the CUDA device");
  }
  int num_sms = 0;
  if ((rc = select_device(device_id, &num_sms)) != TG_OK) return rc;
  const TgTensorDesc* in[2] = {K, V};
  for (int i = 0; i < 2; ++i) {
    p.x[i] = reinterpret_cast<const void*>(in[i]->ptr);
    p.tok_pitch[i] = in[i]->strides[0];
    p.head_pitch[i] = in[i]->strides[1];
  }
  p.tokens = static_cast<int32_t>(T);
  p.tiles = static_cast<int32_t>(tiles);
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(blocks)), block(kWriteThreads);
  cudaError_t e;
  if (K->dtype == TG_BF16)
    e = D == 128 ? launch_pdl(tg_kv_cache_write_kernel<__nv_bfloat16, 128>, grid, block, 0, st, p)
                 : launch_pdl(tg_kv_cache_write_kernel<__nv_bfloat16, 64>, grid, block, 0, st, p);
  else
    e = D == 128 ? launch_pdl(tg_kv_cache_write_kernel<__half, 128>, grid, block, 0, st, p)
                 : launch_pdl(tg_kv_cache_write_kernel<__half, 64>, grid, block, 0, st, p);
  return launch_status(e, "kv_cache_write");
}

extern "C" TG_API int32_t tg_kv_cache_read(const TgTensorDesc* Ko, const TgTensorDesc* Vo, const TgTensorDesc* Kc, const TgTensorDesc* Vc,
                                           const TgTensorDesc* Ks, const TgTensorDesc* Vs, const TgTensorDesc* block_table,
                                           const TgTensorDesc* seq_lens, int32_t device_id, uint64_t stream) {
  ReadParams p = {};
  int32_t rc;
  if ((rc = check_cache(&p.c, Kc, Vc, Ks, Vs, block_table, seq_lens, nullptr)) != TG_OK) return rc;
  if (Ko == nullptr || Vo == nullptr) return api_fail(TG_ERR_NULL, "an output descriptor is null");
  if (!is_16bit(Ko->dtype)) return api_fail(TG_ERR_DTYPE, "the outputs must be bf16 or f16");
  if (Ko->ndim != 4) return api_fail(TG_ERR_ARGS, "the outputs must be [seqs, max_len, heads, head_dim]");
  const int64_t max_len = Ko->shape[1];
  const int64_t shape[4] = {p.c.seqs, max_len, p.c.heads, p.c.dim};
  if ((rc = check_dense_nd(Ko, "k output: [seqs, max_len, heads, head_dim], contiguous, 16-byte aligned", Ko->dtype, 4, shape, 16)) != TG_OK) return rc;
  if ((rc = check_dense_nd(Vo, "v output: [seqs, max_len, heads, head_dim], contiguous, 16-byte aligned", Ko->dtype, 4, shape, 16)) != TG_OK) return rc;
  if (max_len > 0x7fffff80 || p.c.heads > 32767 || p.c.seqs > 65535) return api_fail(TG_ERR_ARGS, "at most 65535 sequences, 32767 heads and 2^31 - 128 rows");
  if (p.c.seqs == 0 || max_len == 0) return TG_OK;
  ScopedDevice guard(device_id);
  if (guard.err != cudaSuccess) {
    cudaGetLastError();
    return api_fail(TG_ERR_DEVICE, "cannot select the CUDA device");
  }
  int num_sms = 0;
  if ((rc = select_device(device_id, &num_sms)) != TG_OK) return rc;
  p.out[0] = reinterpret_cast<void*>(Ko->ptr);
  p.out[1] = reinterpret_cast<void*>(Vo->ptr);
  p.max_len = static_cast<int32_t>(max_len);
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const dim3 grid(static_cast<unsigned>((max_len + kPage - 1) / kPage), p.c.heads * 2, p.c.seqs), block(256);
  cudaError_t e;
  if (Ko->dtype == TG_BF16)
    e = p.c.dim == 128 ? launch_pdl(tg_kv_cache_read_kernel<__nv_bfloat16, 128>, grid, block, 0, st, p)
                       : launch_pdl(tg_kv_cache_read_kernel<__nv_bfloat16, 64>, grid, block, 0, st, p);
  else
    e = p.c.dim == 128 ? launch_pdl(tg_kv_cache_read_kernel<__half, 128>, grid, block, 0, st, p)
                       : launch_pdl(tg_kv_cache_read_kernel<__half, 64>, grid, block, 0, st, p);
  return launch_status(e, "kv_cache_read");
}
