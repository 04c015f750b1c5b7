// Shared by the decoder operators around the GEMMs (RMS norm, rotary positions, 8-bit key / value cache, attention):
// argument checks of their C entry points, the walk over ragged batches, power-of-two cache scales and exact
// rotary angles.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <stdint.h>

#include <type_traits>

#include "tg_internal.h"
#include "tg_ptx.cuh"
#include "tg_quant_common.cuh"

namespace tg {

constexpr int kPage = 128;                // tokens of a cache page: one scale per (page, head) for keys and for values
constexpr int kScaleLo = -60, kScaleHi = 60;  // exponents of a cache scale

// Makes `dev` current for the scope.
struct ScopedDevice {
  int prev = -1;
  bool changed = false;
  cudaError_t err = cudaSuccess;
  explicit ScopedDevice(int dev) {
    err = cudaGetDevice(&prev);
    if (err == cudaSuccess && prev != dev) {
      err = cudaSetDevice(dev);
      changed = (err == cudaSuccess);
    }
  }
  ~ScopedDevice() {
    if (changed) cudaSetDevice(prev);
  }
  ScopedDevice(const ScopedDevice&) = delete;
  ScopedDevice& operator=(const ScopedDevice&) = delete;
};

// ------------------------------------------------------------------------------------------ host-side checks
inline bool is_16bit(int32_t d) { return d == TG_BF16 || d == TG_F16; }

// [rows, heads, dim] in 16 bits: the last dimension dense, rows and heads at any pitch that keeps 16-byte alignment
inline int32_t check_heads(const TgTensorDesc* t, const char* what, int64_t rows, int64_t heads, int64_t dim, int32_t dtype) {
  if (t == nullptr) return api_fail(TG_ERR_NULL, what);
  if (t->ndim != 3 || t->shape[0] != rows || t->shape[1] != heads || t->shape[2] != dim) return api_fail(TG_ERR_ARGS, what);
  if (t->dtype != dtype) return api_fail(TG_ERR_DTYPE, what);
  if (dim > 1 && t->strides[2] != 1) return api_fail(TG_ERR_ARGS, what);
  if (rows > 0 && heads > 0) {
    if (t->ptr == 0) return api_fail(TG_ERR_NULL, what);
    if ((t->ptr & 15u) || (rows > 1 && (t->strides[0] & 7)) || (heads > 1 && (t->strides[1] & 7))) return api_fail(TG_ERR_ALIGN, what);
    if (t->strides[0] < 0 || t->strides[1] < 0) return api_fail(TG_ERR_ARGS, what);
  }
  return TG_OK;
}

// The same for a tensor that is written: no element of it lies on another one.
inline int32_t check_heads_out(const TgTensorDesc* t, const char* what, int64_t rows, int64_t heads, int64_t dim, int32_t dtype) {
  const int32_t rc = check_heads(t, what, rows, heads, dim, dtype);
  if (rc != TG_OK || rows < 1 || heads < 1) return rc;
  int64_t n[2] = {rows, heads}, pitch[2] = {t->strides[0], t->strides[1]};
  if (n[0] == 1 || (n[1] > 1 && pitch[0] > pitch[1])) {  // the smaller pitch, or the dimension of one, last
    n[0] = heads, n[1] = rows;
    pitch[0] = t->strides[1], pitch[1] = t->strides[0];
  }
  int64_t extent = dim;
  for (int i = 0; i < 2; ++i) {
    if (n[i] == 1) continue;
    if (pitch[i] < extent) return api_fail(TG_ERR_ARGS, "a tensor that is written must not overlap itself");
    extent += (n[i] - 1) * pitch[i];
  }
  return TG_OK;
}

// An output that takes its input's place: every head on itself.
inline int32_t check_heads_place(const TgTensorDesc* out, const TgTensorDesc* in) {
  if (out->ptr != in->ptr || in->shape[0] < 1) return TG_OK;
  if ((in->shape[0] > 1 && out->strides[0] != in->strides[0]) || (in->shape[1] > 1 && out->strides[1] != in->strides[1]))
    return api_fail(TG_ERR_ARGS, "an output in the place of its input must have the same pitches");
  return TG_OK;
}

inline int32_t check_dense_nd(const TgTensorDesc* t, const char* what, int32_t dtype, int nd, const int64_t* shape, unsigned align) {
  if (t == nullptr) return api_fail(TG_ERR_NULL, what);
  if (t->dtype != dtype) return api_fail(TG_ERR_DTYPE, what);
  if (t->ndim != nd) return api_fail(TG_ERR_ARGS, what);
  bool empty = false;
  for (int d = 0; d < nd; ++d) {
    if (t->shape[d] != shape[d] || t->shape[d] < 0) return api_fail(TG_ERR_ARGS, what);
    empty = empty || t->shape[d] == 0;
  }
  int64_t expect = 1;
  for (int d = nd - 1; d >= 0 && !empty; --d) {
    if (t->shape[d] > 1 && t->strides[d] != expect) return api_fail(TG_ERR_ARGS, what);
    expect *= t->shape[d];
  }
  if (!empty && t->ptr == 0) return api_fail(TG_ERR_NULL, what);
  if (t->ptr & (align - 1)) return api_fail(TG_ERR_ALIGN, what);
  return TG_OK;
}

// The four tensors of a cache and the tables that say which pages a sequence has.
struct CacheView {
  uint8_t* k = nullptr;    // [pages, heads, kPage, dim]
  uint8_t* v = nullptr;    // [pages, heads, dim, kPage]
  float* ks = nullptr;     // [pages, heads]
  float* vs = nullptr;
  const int32_t* table = nullptr;  // [seqs, table_pitch]
  const int32_t* seq_lens = nullptr;
  const int32_t* cu = nullptr;  // [seqs + 1] or null: one new token per sequence
  int64_t table_pitch = 0;
  int32_t pages = 0, heads = 0, dim = 0, seqs = 0, max_pages = 0;
};

inline int32_t check_cache(CacheView* c, const TgTensorDesc* K, const TgTensorDesc* V, const TgTensorDesc* Ks, const TgTensorDesc* Vs,
                           const TgTensorDesc* table, const TgTensorDesc* lens, const TgTensorDesc* cu) {
  if (K == nullptr || table == nullptr || lens == nullptr) return api_fail(TG_ERR_NULL, "a cache descriptor is null");
  if (K->ndim != 4) return api_fail(TG_ERR_ARGS, "the key cache must be [pages, heads, 128, head_dim]");
  const int64_t pages = K->shape[0], heads = K->shape[1], dim = K->shape[3];
  if (K->shape[2] != kPage) return api_fail(TG_ERR_ARGS, "a cache page holds 128 tokens");
  if (dim != 64 && dim != 128) return api_fail(TG_ERR_ARGS, "head_dim of the cache must be 64 or 128");
  if (heads < 1 || pages < 0 || pages * heads > (int64_t(1) << 24) - 1)
    return api_fail(TG_ERR_ARGS, "the cache needs at least one head and fewer than 2^24 (page, head) blocks");
  const int64_t ks[4] = {pages, heads, kPage, dim}, vs[4] = {pages, heads, dim, kPage}, ss[2] = {pages, heads};
  int32_t rc;
  if ((rc = check_dense_nd(K, "key cache: float8_e4m3fn [pages, heads, 128, head_dim], contiguous, 16-byte aligned", TG_F8E4M3, 4, ks, 16)) != TG_OK) return rc;
  if ((rc = check_dense_nd(V, "value cache: float8_e4m3fn [pages, heads, head_dim, 128], contiguous, 16-byte aligned", TG_F8E4M3, 4, vs, 16)) != TG_OK) return rc;
  if ((rc = check_dense_nd(Ks, "key scales: f32 [pages, heads], contiguous", TG_F32, 2, ss, 4)) != TG_OK) return rc;
  if ((rc = check_dense_nd(Vs, "value scales: f32 [pages, heads], contiguous", TG_F32, 2, ss, 4)) != TG_OK) return rc;
  if (lens->ndim != 1) return api_fail(TG_ERR_ARGS, "seq_lens must be [seqs]");
  const int64_t seqs = lens->shape[0];
  const int64_t ls[1] = {seqs}, cs[1] = {seqs + 1};
  if (seqs > (1 << 20)) return api_fail(TG_ERR_ARGS, "at most 2^20 sequences");
  if ((rc = check_dense_nd(lens, "seq_lens: int32 [seqs], contiguous", TG_I32, 1, ls, 4)) != TG_OK) return rc;
  if (cu != nullptr && (rc = check_dense_nd(cu, "cu_seqlens: int32 [seqs + 1], contiguous", TG_I32, 1, cs, 4)) != TG_OK) return rc;
  if (table->dtype != TG_I32) return api_fail(TG_ERR_DTYPE, "block_table must be int32");
  if (table->ndim != 2 || table->shape[0] != seqs || (table->shape[1] > 1 && table->strides[1] != 1) || table->strides[0] < 0)
    return api_fail(TG_ERR_ARGS, "block_table must be [seqs, pages per sequence] with dense rows");
  if (table->shape[1] > (1 << 24) - 1) return api_fail(TG_ERR_ARGS, "block_table rows are limited to 2^24 - 1 pages");
  if (seqs > 0 && table->shape[1] > 0 && table->ptr == 0) return api_fail(TG_ERR_NULL, "block_table pointer is null");
  if (table->ptr & 3u) return api_fail(TG_ERR_ALIGN, "block_table must be 4-byte aligned");
  c->k = reinterpret_cast<uint8_t*>(K->ptr);
  c->v = reinterpret_cast<uint8_t*>(V->ptr);
  c->ks = reinterpret_cast<float*>(Ks->ptr);
  c->vs = reinterpret_cast<float*>(Vs->ptr);
  c->table = reinterpret_cast<const int32_t*>(table->ptr);
  c->seq_lens = reinterpret_cast<const int32_t*>(lens->ptr);
  c->cu = cu ? reinterpret_cast<const int32_t*>(cu->ptr) : nullptr;
  c->table_pitch = table->strides[0];
  c->pages = static_cast<int32_t>(pages);
  c->heads = static_cast<int32_t>(heads);
  c->dim = static_cast<int32_t>(dim);
  c->seqs = static_cast<int32_t>(seqs);
  c->max_pages = static_cast<int32_t>(table->shape[1]);
  return TG_OK;
}

// Launch with programmatic stream serialization: the kernel's blocks may be scheduled while the kernel in front drains;
// each of these kernels calls griddep_wait() before it touches global memory.
template <typename... P, typename... A>
inline cudaError_t launch_pdl(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = api_pdl() ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

// ------------------------------------------------------------------------------------------ device side
// New tokens of sequence b: rows [lo, hi) of the batch.  Offsets that a caller got wrong stay inside the batch.
__device__ __forceinline__ void new_rows(const int32_t* cu, int b, int tokens, int& lo, int& hi) {
  lo = cu ? min(max(cu[b], 0), tokens) : b;
  hi = cu ? min(max(cu[b + 1], lo), tokens) : b + 1;
}

// Ragged tiles are numbered without a prefix sum over the batch: sequence b owns the numbers from cu[b] / div + per_seq * b
// on, which leaves it floor(n / div) + per_seq or more of them (unused ones exit at once).  Returns the sequence that owns
// `tile` and its first number; called by whole warps, one 32-way search step for each factor of 32 in the batch.
__device__ __forceinline__ int find_sequence(const int32_t* cu, int seqs, int tile, int div, int per_seq, int& first) {
  const int lane = threadIdx.x & 31;
  int lo = 0, n = seqs;
  while (n > 1) {
    const int step = (n + 31) >> 5, at = lo + lane * step;
    const bool below = lane * step < n && (cu ? max(cu[at], 0) : at) / div + per_seq * at <= tile;
    const int count = max(__popc(__ballot_sync(0xffffffffu, below)), 1);
    const int end = lo + n;
    lo += (count - 1) * step;
    n = min(step, end - lo);
  }
  first = (cu ? max(cu[lo], 0) : lo) / div + per_seq * lo;
  return lo;
}

// Smallest power of two s with amax / s <= 448, exponent in [kScaleLo, kScaleHi]: 448 = 1.75 * 2^8.
__device__ __forceinline__ float cache_scale(float amax) {
  const uint32_t b = __float_as_uint(amax);
  const int e = static_cast<int>(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return __uint_as_float(static_cast<uint32_t>(min(max(e, kScaleLo), kScaleHi) + 127) << 23);
}
__device__ __forceinline__ float pow2_reciprocal(float s) { return __uint_as_float((254u << 23) - __float_as_uint(s)); }

// Rotary angles.  A frequency is kept as a 64-bit binary fraction of a turn per position, so that position * fraction
// modulo 2^64 IS the angle modulo one turn: exact for every position, near or far, where a 32-bit product loses 2^-24 of
// the angle itself (a radian at position 10^7).  What remains is the top 32 bits as a signed fraction of a turn.
__device__ __forceinline__ uint64_t turn_fraction(double inv_freq) {
  const double turns = inv_freq * 0.15915494309189533577;  // 1 / (2 pi)
  const double part = turns - floor(turns);
  return static_cast<uint64_t>(__double2ull_rn(part * 18446744073709551616.0));
}
__device__ __forceinline__ float2 cos_sin_at(uint64_t fraction, int64_t position, float magnitude) {
  const int32_t top = static_cast<int32_t>((fraction * static_cast<uint64_t>(position)) >> 32);
  // |angle| <= pi: the hardware sine and cosine are within 2^-21 there, far below half a step of the 16-bit outputs
  const float angle = static_cast<float>(top) * 1.4629180792671596e-9f;  // 2 pi / 2^32
  return make_float2(__cosf(angle) * magnitude, __sinf(angle) * magnitude);
}

template <typename T>
__device__ __forceinline__ uint32_t pack_pair(float a, float b) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

// One pair turned: written out so that every kernel rounds alike.
__device__ __forceinline__ float turn_first(float x, float y, float2 cs) { return __fmaf_rn(x, cs.x, -__fmul_rn(y, cs.y)); }
__device__ __forceinline__ float turn_second(float x, float y, float2 cs) { return __fmaf_rn(y, cs.x, __fmul_rn(x, cs.y)); }

// Turns 8 pairs.  Half layout: a holds elements i .. i + 7 of the head, b their partners i + rotary / 2 ..; interleaved:
// a and b hold 16 neighbouring elements and pairs sit side by side.  Both come back rounded to T.
template <typename T>
__device__ __forceinline__ void rotate_unit(uint4& a, uint4& b, const float2 (&cs)[8], bool interleaved) {
  uint32_t* wa = reinterpret_cast<uint32_t*>(&a);
  uint32_t* wb = reinterpret_cast<uint32_t*>(&b);
  if (interleaved) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 x = unpack_pair<T>(wa[i]), y = unpack_pair<T>(wb[i]);
      wa[i] = pack_pair<T>(turn_first(x.x, x.y, cs[i]), turn_second(x.x, x.y, cs[i]));
      wb[i] = pack_pair<T>(turn_first(y.x, y.y, cs[i + 4]), turn_second(y.x, y.y, cs[i + 4]));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 x = unpack_pair<T>(wa[i]), y = unpack_pair<T>(wb[i]);
      const float2 c0 = cs[2 * i], c1 = cs[2 * i + 1];
      wa[i] = pack_pair<T>(turn_first(x.x, y.x, c0), turn_first(x.y, y.y, c1));
      wb[i] = pack_pair<T>(turn_second(x.x, y.x, c0), turn_second(x.y, y.y, c1));
    }
  }
}

// Where the two 8-element vectors of unit w of a head (dim / 16 units) start, and its first pair (-1: not rotated).
__device__ __forceinline__ void unit_offsets(int w, int rotary, bool interleaved, int& oa, int& ob, int& pair) {
  if (w * 16 < rotary) {
    oa = interleaved ? w * 16 : w * 8;
    ob = interleaved ? w * 16 + 8 : rotary / 2 + w * 8;
    pair = w * 8;
  } else {
    oa = w * 16;
    ob = oa + 8;
    pair = -1;
  }
}

}  // namespace tg
