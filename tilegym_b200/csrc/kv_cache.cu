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

// ------------------------------------------------------------------------------------------ rotation by warps
struct RopeHeads {
  const void* in;
  void* out;
  int64_t in_tok, in_head, out_tok, out_head;  // pitches in elements
  int32_t heads;
};

constexpr int kMaxPairs = 256;

// A warp turns heads of one token.  A lane keeps one unit (16 elements, 8 pairs) of the head for all heads that it comes to,
// so the cosines and sines stay in registers: no shared memory, no barrier, and the loads of four heads are in flight at
// once.  `parts` warps share a token's heads where there are few tokens.  Bound: HBM; 8191 tokens x 40 heads x 128 elements
// (168 MB) measured 30 us (5.6 TB/s), 37 with a block per token and the angles in shared memory.
template <typename T>
__device__ __forceinline__ void rotate_token(const RopeHeads& q, const RopeHeads& k, int64_t tok, int64_t pos, int part, int parts, int units,
                                             const RopeParams& r) {
  const int lane = threadIdx.x & 31;
  const int per = 32 / units;  // heads side by side in the warp
  const int sub = lane / units, w = lane - sub * units;
  const bool inter = r.interleaved != 0;
  int oa, ob, pair;
  unit_offsets(w, r.rotary, inter, oa, ob, pair);
  float2 cs[8];
  if (pair >= 0) {
#pragma unroll
    for (int i = 0; i < 8; ++i) cs[i] = cos_sin_at(turn_fraction(r.inv_freq[pair + i]), pos, r.magnitude);
  }
  const int total = sub < per ? q.heads + k.heads : 0;
  const T* qi = static_cast<const T*>(q.in) + tok * q.in_tok;
  const T* ki = static_cast<const T*>(k.in) + tok * k.in_tok;
  T* qo = static_cast<T*>(q.out) + tok * q.out_tok;
  T* ko = static_cast<T*>(k.out) + tok * k.out_tok;
  const int step = per * parts;
  for (int h0 = part * per + sub; h0 < total; h0 += 4 * step) {
    uint4 a[4], b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int h = h0 + i * step;
      if (h < total) {
        const T* src = h < q.heads ? qi + h * q.in_head : ki + (h - q.heads) * k.in_head;
        a[i] = *reinterpret_cast<const uint4*>(src + oa);
        b[i] = *reinterpret_cast<const uint4*>(src + ob);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int h = h0 + i * step;
      if (h < total) {
        if (pair >= 0) rotate_unit<T>(a[i], b[i], cs, inter);
        T* dst = h < q.heads ? qo + h * q.out_head : ko + (h - q.heads) * k.out_head;
        *reinterpret_cast<uint4*>(dst + oa) = a[i];
        *reinterpret_cast<uint4*>(dst + ob) = b[i];
      }
    }
  }
}

// Warps that share a token: as many as it takes to have 16 for every SM, no more than there are turns.
int warps_per_token(int64_t tokens, int heads, int units, int num_sms) {
  const int per = 32 / units, turns = (heads + per - 1) / per;
  const int64_t want = (16ll * num_sms + tokens - 1) / tokens;
  return static_cast<int>(want < 1 ? 1 : want > turns ? turns : want);
}

// ------------------------------------------------------------------------------------------ apply_rope
struct ApplyRopeParams {
  RopeHeads q, k;
  RopeParams rope;
  const void* positions;
  int32_t positions64, tokens, units, parts;
};

constexpr int kRopeThreads = 128;

template <typename T>
__global__ void __launch_bounds__(kRopeThreads) tg_apply_rope_kernel(const ApplyRopeParams p) {
  griddep_wait();
  griddep_launch_dependents();
  const int64_t id = static_cast<int64_t>(blockIdx.x) * (kRopeThreads / 32) + (threadIdx.x >> 5);
  const int64_t tok = id / p.parts;
  if (tok >= p.tokens) return;
  const int64_t pos = p.positions64 ? static_cast<const int64_t*>(p.positions)[tok] : static_cast<const int32_t*>(p.positions)[tok];
  rotate_token<T>(p.q, p.k, tok, pos, static_cast<int>(id - tok * p.parts), p.parts, p.units, p.rope);
}

// ------------------------------------------------------------------------------------------ kv_cache_write
struct WriteParams {
  CacheView c;
  const void* x[2];  // new keys, new values [tokens, heads, dim]
  int64_t tok_pitch[2], head_pitch[2];
  RopeParams rope;  // inv_freq null: keys are written as they come
  RopeHeads q;      // queries rotated beside the keys; heads 0: none
  int32_t tokens, tiles, cache_blocks, parts;
};

constexpr int kWriteThreads = 256;

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

// The first t0 tokens of a block move from one scale to another (f = old / new); `n` threads share the work.
template <int DIM>
__device__ __forceinline__ void rescale_block(uint8_t* dst, bool is_v, int t0, float f, int i0, int n) {
  if (is_v) {
#pragma unroll 4
    for (int i = i0; i < DIM * (kPage / 16); i += n) {
      const int t = (i % (kPage / 16)) * 16;
      if (t >= t0) continue;
      uint4* at = reinterpret_cast<uint4*>(dst) + i;
      uint4 w = *at;
      w.x = merge_low(w.x, requantise4(w.x, f), t0 - t);
      w.y = merge_low(w.y, requantise4(w.y, f), t0 - t - 4);
      w.z = merge_low(w.z, requantise4(w.z, f), t0 - t - 8);
      w.w = merge_low(w.w, requantise4(w.w, f), t0 - t - 12);
      *at = w;
    }
  } else {
#pragma unroll 4
    for (int i = i0; i < t0 * (DIM / 16); i += n) {
      uint4* at = reinterpret_cast<uint4*>(dst) + i;
      const uint4 w = *at;
      *at = make_uint4(requantise4(w.x, f), requantise4(w.y, f), requantise4(w.z, f), requantise4(w.w, f));
    }
  }
}

// What a tile number stands for: a page of a sequence and the tokens of it that are new.
struct WriteTile {
  int page, phys, t0, t1;
  int64_t row0;  // batch row of the page's token 0
};
__device__ __forceinline__ bool locate_write(const WriteParams& p, int tile, WriteTile& w) {
  int first, lo, hi;
  const int b = find_sequence(p.c.cu, p.c.seqs, tile, kPage, 2, first);
  new_rows(p.c.cu, b, p.tokens, lo, hi);
  const int len = p.c.seq_lens[b], start = len - (hi - lo);  // positions start .. len - 1 are new
  if (hi <= lo || len <= 0 || tile < first) return false;
  w.page = max(start, 0) / kPage + (tile - first);
  if (w.page * kPage >= len || w.page >= p.c.max_pages) return false;
  w.phys = p.c.table[b * p.c.table_pitch + w.page];
  if (w.phys < 0 || w.phys >= p.c.pages) return false;
  w.t0 = max(start - w.page * kPage, 0);
  w.t1 = min(len - w.page * kPage, kPage);
  w.row0 = static_cast<int64_t>(lo) + w.page * kPage - start;
  return true;
}

// Many new tokens: a block owns one (page of a sequence, head) of the keys or of the values, so nobody else touches that
// block's scale or bytes.  The new values stay in registers between the maximum and the rounding; values are turned to
// [dim][token] in shared memory four by four bytes (words of four elements in, 16 tokens of four elements out, swizzled by
// the token group so that neither side meets a bank twice).  Bound: HBM and the 8-bit conversions; a ragged prefill with its
// queries (347 MB) measured 63 us (5.5 TB/s), 128 with 128 threads per block and byte stores.
template <typename T, int DIM>
__device__ __forceinline__ void write_tile(const WriteParams& p, const WriteTile& at, int head, bool is_v, uint64_t* fraction, uint32_t* words,
                                           float* red) {
  constexpr int kUnits = DIM / 16;                      // units of 16 elements per token
  constexpr int kPer = kPage * kUnits / kWriteThreads;  // units per thread when a whole page is new
  constexpr int kRow = DIM / 4;                         // words of a token in shared memory
  const int64_t block = static_cast<int64_t>(at.phys) * p.c.heads + head;
  const T* x = static_cast<const T*>(p.x[is_v]) + head * p.head_pitch[is_v];
  const int t0 = at.t0, t1 = at.t1, count = (t1 - t0) * kUnits;
  const bool rope = !is_v && p.rope.inv_freq != nullptr;
  const bool inter = p.rope.interleaved != 0;
  const int rotary = rope ? p.rope.rotary : 0;
  int oa, ob, pair;  // the same unit of the head for all of a thread's tokens
  unit_offsets(threadIdx.x % kUnits, rotary, inter, oa, ob, pair);
  static_assert(kWriteThreads % kUnits == 0, "");
  const int tt = t0 + threadIdx.x / kUnits;  // and tokens tt, tt + kWriteThreads / kUnits, ..

  uint4 va[kPer], vb[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    va[i] = vb[i] = make_uint4(0, 0, 0, 0);
    if (i * kWriteThreads + static_cast<int>(threadIdx.x) < count) {
      const T* src = x + (at.row0 + tt + i * (kWriteThreads / kUnits)) * p.tok_pitch[is_v];
      va[i] = *reinterpret_cast<const uint4*>(src + oa);
      vb[i] = *reinterpret_cast<const uint4*>(src + ob);
    }
  }
  if (rope) {
    for (int i = threadIdx.x; i < rotary / 2; i += kWriteThreads) fraction[i] = turn_fraction(p.rope.inv_freq[i]);
    __syncthreads();
    if (pair >= 0) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int pos = at.page * kPage + tt + i * (kWriteThreads / kUnits);
        float2 cs[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) cs[j] = cos_sin_at(fraction[pair + j], pos, p.rope.magnitude);
        rotate_unit<T>(va[i], vb[i], cs, inter);  // zeros stay zeros
      }
    }
  }
  uint32_t m2 = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    m2 = absmax_pairs<T>(m2, absmax_pairs<T>(absmax_pairs<T>(va[i].x, va[i].y), absmax_pairs<T>(va[i].z, va[i].w)));
    m2 = absmax_pairs<T>(m2, absmax_pairs<T>(absmax_pairs<T>(vb[i].x, vb[i].y), absmax_pairs<T>(vb[i].z, vb[i].w)));
  }
  const float2 mm = unpack_pair<T>(m2);
  float amax = fmaxf(mm.x, mm.y);
  if (!(amax <= 3.4028234e38f)) {  // an infinity does not count (the packed maximum has passed over NaN)
    amax = 0.f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const uint32_t w[8] = {va[i].x, va[i].y, va[i].z, va[i].w, vb[i].x, vb[i].y, vb[i].z, vb[i].w};
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float2 f = unpack_pair<T>(w[j]);
        amax = fmaxf(amax, fmaxf(finite_abs(f.x), finite_abs(f.y)));
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = amax;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWriteThreads / 32; ++i) amax = fmaxf(amax, red[i]);
  float s = cache_scale(amax);
  float* scale = (is_v ? p.c.vs : p.c.ks) + block;
  uint8_t* dst = (is_v ? p.c.v : p.c.k) + block * (kPage * DIM);
  if (t0 > 0) {
    const float old = *scale;
    if (old >= s) s = old;
    else rescale_block<DIM>(dst, is_v, t0, old * pow2_reciprocal(s), threadIdx.x, kWriteThreads);
    __syncthreads();  // the scale is read by all before it is written, old bytes are moved before new ones arrive
  }
  if (threadIdx.x == 0) *scale = s;
  const float r = 1.0f / s;  // exact but for a kept scale that is no power of two
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (i * kWriteThreads + static_cast<int>(threadIdx.x) >= count) continue;
    const int t = tt + i * (kWriteThreads / kUnits);
    const uint32_t w[8] = {va[i].x, va[i].y, va[i].z, va[i].w, vb[i].x, vb[i].y, vb[i].z, vb[i].w};
    uint32_t q[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f0 = unpack_pair<T>(w[2 * j]), f1 = unpack_pair<T>(w[2 * j + 1]);
      q[j] = q8_cast2<kQ8E4M3>(f0.x * r, f0.y * r, 0.f, 0.f) | (q8_cast2<kQ8E4M3>(f1.x * r, f1.y * r, 0.f, 0.f) << 16);
    }
    if (is_v) {
      const int swz = ((t >> 4) << 2) & (kRow - 1);
      *reinterpret_cast<uint2*>(words + t * kRow + ((oa >> 2) ^ swz)) = make_uint2(q[0], q[1]);
      *reinterpret_cast<uint2*>(words + t * kRow + ((ob >> 2) ^ swz)) = make_uint2(q[2], q[3]);
    } else {
      *reinterpret_cast<uint2*>(dst + t * DIM + oa) = make_uint2(q[0], q[1]);
      *reinterpret_cast<uint2*>(dst + t * DIM + ob) = make_uint2(q[2], q[3]);
    }
  }
  if (!is_v) return;
  __syncthreads();
  for (int i = threadIdx.x; i < kRow * (kPage / 16); i += kWriteThreads) {
    const int tg = i & 7, dw = i >> 3, t = tg * 16;  // four elements from 4 dw, sixteen tokens from t
    if (t >= t1 || t + 16 <= t0) continue;
    const int col = dw ^ ((tg << 2) & (kRow - 1));
    uint32_t o[4][4];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = words[(t + g * 4 + j) * kRow + col];
      const uint32_t ab_lo = __byte_perm(w[0], w[1], 0x5140), ab_hi = __byte_perm(w[0], w[1], 0x7362);
      const uint32_t cd_lo = __byte_perm(w[2], w[3], 0x5140), cd_hi = __byte_perm(w[2], w[3], 0x7362);
      o[0][g] = __byte_perm(ab_lo, cd_lo, 0x5410);
      o[1][g] = __byte_perm(ab_lo, cd_lo, 0x7632);
      o[2][g] = __byte_perm(ab_hi, cd_hi, 0x5410);
      o[3][g] = __byte_perm(ab_hi, cd_hi, 0x7632);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      uint8_t* to = dst + (dw * 4 + e) * kPage + t;
      if (t >= t0 && t + 16 <= t1) {
        *reinterpret_cast<uint4*>(to) = make_uint4(o[e][0], o[e][1], o[e][2], o[e][3]);
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (t + j >= t0 && t + j < t1) to[j] = static_cast<uint8_t>(o[e][j >> 2] >> (8 * (j & 3)));
      }
    }
  }
}

// Few new tokens (a decode step): a warp owns the (page, head), a lane DIM / 32 neighbouring elements, and the tokens are
// gone through twice, for the maximum and for the bytes.  Latency: 128 sequences of a decode batch, 8 heads, with their
// queries measured 5.7 us where no block moves to a larger scale (24.6 with a block per (page, head)); on caches that are not
// in L2 6.8 us, 15 where half of the blocks move and 16 where all do (33 MB of cache, read and written by those warps).
template <typename T, int DIM>
__device__ __forceinline__ void write_append(const WriteParams& p, const WriteTile& at, int head, bool is_v) {
  constexpr int E = DIM / 32;
  const int lane = threadIdx.x & 31, e0 = lane * E;
  const int64_t block = static_cast<int64_t>(at.phys) * p.c.heads + head;
  const T* x = static_cast<const T*>(p.x[is_v]) + head * p.head_pitch[is_v];
  float* scale = (is_v ? p.c.vs : p.c.ks) + block;
  uint8_t* dst = (is_v ? p.c.v : p.c.k) + block * (kPage * DIM);
  const float old = at.t0 > 0 ? *scale : 0.f;
  const bool turns = !is_v && p.rope.inv_freq != nullptr && e0 < p.rope.rotary;
  const bool inter = p.rope.interleaved != 0;
  const int half = p.rope.rotary / 2;
  uint64_t fraction[E];
  if (turns) {
#pragma unroll
    for (int j = 0; j < E; ++j) fraction[j] = turn_fraction(p.rope.inv_freq[inter ? (e0 + j) >> 1 : (e0 + j) % half]);
  }
  auto token = [&](int t, float (&v)[E]) {
    const T* src = x + (at.row0 + t) * p.tok_pitch[is_v];
    uint32_t w[E / 2];
#pragma unroll
    for (int j = 0; j < E / 2; ++j) w[j] = *reinterpret_cast<const uint32_t*>(src + e0 + 2 * j);
#pragma unroll
    for (int j = 0; j < E / 2; ++j) {
      const float2 f = unpack_pair<T>(w[j]);
      v[2 * j] = f.x;
      v[2 * j + 1] = f.y;
    }
    if (turns) {
      float o[E];
      const int64_t pos = static_cast<int64_t>(at.page) * kPage + t;
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const float2 cs = cos_sin_at(fraction[j], pos, p.rope.magnitude);
        const bool second = inter ? (j & 1) : e0 >= half;
        const float other = inter ? v[j ^ 1] : static_cast<float>(src[second ? e0 + j - half : e0 + j + half]);
        o[j] = second ? turn_second(other, v[j], cs) : turn_first(v[j], other, cs);
      }
#pragma unroll
      for (int j = 0; j < E; ++j) v[j] = static_cast<float>(static_cast<T>(o[j]));
    }
  };
  float amax = 0.f, v[E];
  for (int t = at.t0; t < at.t1; ++t) {
    token(t, v);
#pragma unroll
    for (int j = 0; j < E; ++j) amax = fmaxf(amax, finite_abs(v[j]));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  float s = cache_scale(amax);
  if (at.t0 > 0) {
    if (old >= s) s = old;
    else rescale_block<DIM>(dst, is_v, at.t0, old * pow2_reciprocal(s), lane, 32);
    __syncwarp();
  }
  if (lane == 0) *scale = s;
  const float r = 1.0f / s;  // as in write_tile
  for (int t = at.t0; t < at.t1; ++t) {
    if (at.t1 - at.t0 > 1) token(t, v);  // a single token is still in registers
    uint32_t q = q8_cast2<kQ8E4M3>(v[0] * r, v[1] * r, 0.f, 0.f);
    if constexpr (E == 4) q |= q8_cast2<kQ8E4M3>(v[2] * r, v[3] * r, 0.f, 0.f) << 16;
    if (is_v) {
#pragma unroll
      for (int j = 0; j < E; ++j) dst[(e0 + j) * kPage + t] = static_cast<uint8_t>(q >> (8 * j));
    } else if constexpr (E == 4) {
      *reinterpret_cast<uint32_t*>(dst + t * DIM + e0) = q;
    } else {
      *reinterpret_cast<uint16_t*>(dst + t * DIM + e0) = static_cast<uint16_t>(q);
    }
  }
}

template <typename T, int DIM, bool kAppend>
__global__ void __launch_bounds__(kWriteThreads) tg_kv_cache_write_kernel(const __grid_constant__ WriteParams p) {
  griddep_wait();
  griddep_launch_dependents();
  const int warp = threadIdx.x >> 5;
  if (static_cast<int>(blockIdx.x) < p.cache_blocks) {
    WriteTile at;
    if constexpr (kAppend) {
      const int id = blockIdx.x * (kWriteThreads / 32) + warp, unit = id >> 1;
      const int head = unit % p.c.heads, tile = unit / p.c.heads;
      if (tile < p.tiles && locate_write(p, tile, at)) write_append<T, DIM>(p, at, head, id & 1);
    } else {
      __shared__ __align__(16) uint32_t words[kPage * DIM / 4];
      __shared__ uint64_t fraction[DIM / 2];
      __shared__ float red[kWriteThreads / 32];
      const int unit = blockIdx.x >> 1;
      if (locate_write(p, unit / p.c.heads, at)) write_tile<T, DIM>(p, at, unit % p.c.heads, blockIdx.x & 1, fraction, words, red);
    }
    return;
  }
  // queries
  const int64_t id = (static_cast<int64_t>(blockIdx.x) - p.cache_blocks) * (kWriteThreads / 32) + warp;
  const int64_t tok = id / p.parts;
  if (tok >= p.tokens) return;
  int first, lo, hi;
  // a row belongs to the last sequence that starts at or before it, if that reaches so far
  const int b = find_sequence(p.c.cu, p.c.seqs, static_cast<int>(tok), 1, 0, first);
  new_rows(p.c.cu, b, p.tokens, lo, hi);
  if (tok < lo || tok >= hi) return;
  const RopeHeads none = {};
  rotate_token<T>(p.q, none, tok, static_cast<int64_t>(p.c.seq_lens[b]) - hi + tok, static_cast<int>(id - tok * p.parts), p.parts, DIM / 16, p.rope);
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

template <typename T>
__device__ __forceinline__ uint4 eight_values(uint32_t a, uint32_t b, float s) {
  const float2 f0 = e4m3_pair(a), f1 = e4m3_pair(a >> 16), f2 = e4m3_pair(b), f3 = e4m3_pair(b >> 16);
  return make_uint4(pack_pair<T>(f0.x * s, f0.y * s), pack_pair<T>(f1.x * s, f1.y * s), pack_pair<T>(f2.x * s, f2.y * s), pack_pair<T>(f3.x * s, f3.y * s));
}

// A block turns one (page of a sequence, head) back into 16 bits; rows behind the sequence's length get zeros.  Values are
// turned from [dim][token] in shared memory: a thread takes four tokens of eight elements (words swizzled by the element
// group, so that a warp's reads meet every bank once) and transposes them four by four bytes.  Bound: HBM; 12 sequences of
// up to 8192 tokens, 8 heads of 128 (473 MB) measured 79 us (6.0 TB/s), 162 with single bytes from shared memory.
template <typename T, int DIM>
__global__ void __launch_bounds__(256) tg_kv_cache_read_kernel(const __grid_constant__ ReadParams p) {
  __shared__ __align__(16) uint32_t words[DIM * kPage / 4];
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
  constexpr int kOct = DIM / 8;
  if (!is_v || live == 0) {
    // 8 elements of a row per step
#pragma unroll 4
    for (int i = threadIdx.x; i < rows * kOct; i += 256) {
      const int t = i / kOct, d = (i % kOct) * 8;
      uint4 o = make_uint4(0, 0, 0, 0);
      if (t < live) {
        const uint2 w = *reinterpret_cast<const uint2*>(src + t * DIM + d);
        o = eight_values<T>(w.x, w.y, s);
      }
      __stcs(reinterpret_cast<uint4*>(out + t * pitch + d), o);
    }
    return;
  }
#pragma unroll 4
  for (int i = threadIdx.x; i < DIM * (kPage / 16); i += 256) {
    const int d = i >> 3, c = (i & 7) * 4, swz = (d >> 3) * 2;
    const uint4 w = reinterpret_cast<const uint4*>(src)[i];
    *reinterpret_cast<uint2*>(words + d * 32 + (c ^ swz)) = make_uint2(w.x, w.y);
    *reinterpret_cast<uint2*>(words + d * 32 + ((c + 2) ^ swz)) = make_uint2(w.z, w.w);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kOct * (kPage / 4); i += 256) {
    const int oct = i % kOct, tq = i / kOct, t = tq * 4;
    if (t >= rows) continue;
    uint32_t half[2][4];  // [elements 0-3, 4-7][token]
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = words[(oct * 8 + g * 4 + j) * 32 + (tq ^ (oct * 2))];
      const uint32_t ab_lo = __byte_perm(w[0], w[1], 0x5140), ab_hi = __byte_perm(w[0], w[1], 0x7362);
      const uint32_t cd_lo = __byte_perm(w[2], w[3], 0x5140), cd_hi = __byte_perm(w[2], w[3], 0x7362);
      half[g][0] = __byte_perm(ab_lo, cd_lo, 0x5410);
      half[g][1] = __byte_perm(ab_lo, cd_lo, 0x7632);
      half[g][2] = __byte_perm(ab_hi, cd_hi, 0x5410);
      half[g][3] = __byte_perm(ab_hi, cd_hi, 0x7632);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (t + j >= rows) break;
      __stcs(reinterpret_cast<uint4*>(out + (t + j) * pitch + oct * 8),
             t + j < live ? eight_values<T>(half[0][j], half[1][j], s) : make_uint4(0, 0, 0, 0));
    }
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
  if (T < 0 || T > (1 << 28)) return api_fail(TG_ERR_ARGS, "too many tokens");
  if (D < 16 || D % 16 != 0 || D > 2 * kMaxPairs) return api_fail(TG_ERR_ARGS, "head_dim must be a multiple of 16 up to 512");
  if (Q->shape[1] < 1 || Q->shape[1] > 65536) return api_fail(TG_ERR_ARGS, "q needs 1 to 65536 heads");
  ApplyRopeParams p = {};
  int32_t rc;
  if ((rc = check_heads(Q, "q: rows of a head dense, pitches and pointer 16-byte aligned", T, Q->shape[1], D, Q->dtype)) != TG_OK) return rc;
  if ((rc = check_heads_out(Qo, "q output: shape and type of q, 16-byte aligned", T, Q->shape[1], D, Q->dtype)) != TG_OK) return rc;
  if ((rc = check_heads_place(Qo, Q)) != TG_OK) return rc;
  p.q = heads_of(Q, Qo);
  if (K != nullptr) {
    if (K->ndim != 3 || K->shape[1] < 1 || K->shape[1] > 65536) return api_fail(TG_ERR_ARGS, "k must be [tokens, heads, head_dim]");
    if ((rc = check_heads(K, "k: tokens, head_dim and type of q, 16-byte aligned", T, K->shape[1], D, Q->dtype)) != TG_OK) return rc;
    if ((rc = check_heads_out(Ko, "k output: shape and type of k, 16-byte aligned", T, K->shape[1], D, Q->dtype)) != TG_OK) return rc;
    if ((rc = check_heads_place(Ko, K)) != TG_OK) return rc;
    p.k = heads_of(K, Ko);
    if (T > 0 && Ko->ptr == Qo->ptr) return api_fail(TG_ERR_ARGS, "q and k must not be written to the same place");
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
  // in place the units behind the rotated ones stay as they are
  const bool in_place = p.q.in == p.q.out && p.k.in == p.k.out;
  p.units = in_place ? p.rope.rotary / 16 : static_cast<int32_t>(D / 16);
  p.tokens = static_cast<int32_t>(T);
  p.parts = warps_per_token(T, p.q.heads + p.k.heads, p.units, num_sms);
  const int64_t blocks = (T * p.parts + kRopeThreads / 32 - 1) / (kRopeThreads / 32);
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(blocks)), block(kRopeThreads);
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
    if ((rc = check_heads_out(Qo, "q output: shape and type of q, 16-byte aligned", T, Q->shape[1], D, K->dtype)) != TG_OK) return rc;
    if ((rc = check_heads_place(Qo, Q)) != TG_OK) return rc;
    p.q = heads_of(Q, Qo);
  }
  if (T == 0 || p.c.seqs == 0) return TG_OK;
  const int64_t tiles = T / kPage + 2 * static_cast<int64_t>(p.c.seqs), units = tiles * p.c.heads * 2;
  // up to four new tokens per sequence on average a warp per block of the cache, from there a thread block
  const bool append = T <= 4 * static_cast<int64_t>(p.c.seqs);
  const int64_t cache_blocks = append ? (units + kWriteThreads / 32 - 1) / (kWriteThreads / 32) : units;
  if (units + T * 64 > 0x7fffffff) return api_fail(TG_ERR_ARGS, "too many tokens and heads for one call");
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
  p.cache_blocks = static_cast<int32_t>(cache_blocks);
  p.parts = Q ? warps_per_token(T, p.q.heads, static_cast<int>(D / 16), num_sms) : 1;
  const int64_t blocks = cache_blocks + (Q ? (T * p.parts + kWriteThreads / 32 - 1) / (kWriteThreads / 32) : 0);
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(blocks)), block(kWriteThreads);
  auto launch = [&](auto tag, auto dim) {
    using E = decltype(tag);
    constexpr int kDim = decltype(dim)::value;
    return append ? launch_pdl(tg_kv_cache_write_kernel<E, kDim, true>, grid, block, 0, st, p)
                  : launch_pdl(tg_kv_cache_write_kernel<E, kDim, false>, grid, block, 0, st, p);
  };
  const std::integral_constant<int, 64> d64;
  const std::integral_constant<int, 128> d128;
  const cudaError_t e = K->dtype == TG_BF16 ? (D == 128 ? launch(__nv_bfloat16(), d128) : launch(__nv_bfloat16(), d64))
                                            : (D == 128 ? launch(__half(), d128) : launch(__half(), d64));
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
