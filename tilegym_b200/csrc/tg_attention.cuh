// Arguments and small device functions of the attention kernels.
#pragma once
#include "tg_decoder_common.cuh"

namespace tg {

struct AttentionParams {
  CacheView c;
  const void* q;  // [tokens, q_heads, dim]
  void* o;
  int64_t q_tok, q_head, o_tok, o_head;  // pitches in elements
  int32_t tokens, q_heads, group;        // group: query heads of one cache head
  float scale;
  int32_t window, sinks;
  int32_t max_q_len;
  int32_t splits;  // many rows: blocks that share the pages of 256 rows
  // workspace: partial results; for few rows of ranges that begin or end inside a unit
  float* part_o;    // few rows: [2 * blocks][rows][dim], many: [blocks][splits][256][dim]
  float2* part_ml;  // the same without dim: reference exponent, sum
  int4* record;     // [blocks]: unit that a block leaves unfinished
  int32_t* status;
  uint32_t wait_limit_us;
};

// Few rows per (sequence, cache head): the cache's bytes are what counts.  37 sequences of 8000 tokens, 8 cache heads of 128,
// with 32 rows each: 160 us, 226 with the kernel for many rows; with 64 rows 481 and 232.
constexpr int kFewRowsMax = 32;
int few_rows_padded(int rows);  // 16 or 32
int few_rows_blocks(int dim, int rows_padded, bool bf16, int num_sms);
uint64_t few_rows_workspace(int dim, int rows_padded, int blocks);
cudaError_t launch_attention_few_rows(const CUtensorMap& tmK, const CUtensorMap& tmV, const AttentionParams& p, int rows_padded,
                                      int blocks, bool bf16, cudaStream_t stream);
// Many rows: the products are what counts.
int64_t many_rows_tiles(int64_t tokens, int64_t seqs, int group);  // pairs of tiles, at most, of all sequences
int many_rows_splits(int64_t tokens, int64_t seqs, int64_t heads, int group, int64_t max_pages, int num_sms);
uint64_t many_rows_workspace(int dim, int64_t blocks, int splits);
cudaError_t launch_attention_many_rows(const CUtensorMap& tmK, const CUtensorMap& tmV, const AttentionParams& p, bool bf16,
                                       cudaStream_t stream);

// ------------------------------------------------------------------------------------------ device side
__device__ __forceinline__ float redux_max(float v) {
  float r;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float exp2_approx(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ void tmem_ld_32x8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_st_32x8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// K-major operand tile with 64-byte rows and the 64-byte swizzle (8-row groups 512 bytes apart): layout type 4.
__device__ __forceinline__ uint64_t make_kmajor_sw64_desc(uint32_t smem_addr) {
  return static_cast<uint64_t>((smem_addr >> 4) & 0x3FFFu) | (1ull << 16) | (static_cast<uint64_t>(512u >> 4) << 32) | (1ull << 46) |
         (4ull << 61);
}
template <int DIM>
__device__ __forceinline__ uint64_t rows_desc(uint32_t smem_addr) {  // rows of DIM bytes
  if constexpr (DIM == 128) return make_kmajor_sw128_desc(smem_addr);
  else return make_kmajor_sw64_desc(smem_addr);
}
// Byte offset of element e of row r in such a tile.
template <int DIM>
__device__ __forceinline__ uint32_t swizzled(int r, int e) {
  const int chunk = e >> 4;
  if constexpr (DIM == 128) return r * 128 + ((chunk ^ (r & 7)) << 4) + (e & 15);
  else return r * 64 + ((chunk ^ ((r >> 1) & 3)) << 4) + (e & 15);
}

// Two values as sums of TERMS pairs of e4m3 values, each `step` times smaller than it is stored beside the one before.
// e4m3 has four significant bits; what a rounding leaves is at most 2^-4 of the value and has a sign again, so two terms
// hold eight bits (a bf16 exactly), three twelve, down to half of the smallest step of the last term.
constexpr float kTermStep = 16.f;
template <int TERMS>
__device__ __forceinline__ void split_e4m3(float lo, float hi, float step, uint32_t (&term)[TERMS]) {
#pragma unroll
  for (int i = 0; i < TERMS; ++i) {
    const __nv_fp8x2_storage_t b = __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
    term[i] = b;
    if (i + 1 == TERMS) break;
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(b, __NV_E4M3);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    lo = (lo - f.x) * step;
    hi = (hi - f.y) * step;
  }
}

// What the new tokens of one sequence see, as a list of pages: the pages of the first tokens that stay visible, then those
// of the windows of all rows.
struct SeqView {
  int lo, n;          // batch rows lo .. lo + n - 1
  int len, pos0;      // tokens in the cache; position of the first new one
  int tiles;          // pages to visit (1, of nothing, where there are rows and no page)
  int sink_tiles, first_page;

  __device__ __forceinline__ int page_of(int t) const { return t < sink_tiles ? t : first_page + t - sink_tiles; }
};
__device__ __forceinline__ SeqView view_sequence(const AttentionParams& p, int b, int first_row, int max_rows) {
  SeqView v;
  int hi;
  new_rows(p.c.cu, b, p.tokens, v.lo, hi);
  const int all = hi - v.lo;
  v.lo += first_row;
  v.n = min(all - first_row, max_rows);
  const int len = p.c.seq_lens[b];
  v.pos0 = len - all + first_row;
  v.len = min(max(len, 0), p.c.max_pages * kPage);
  v.tiles = v.sink_tiles = v.first_page = 0;
  if (v.n <= 0) return v;
  const int last = min(v.len - 1, v.pos0 + v.n - 1);  // last position that any row sees
  if (last < 0) {
    v.tiles = 1;
    v.first_page = p.c.max_pages;  // a page that is not there
    return v;
  }
  const int from = p.window > 0 ? static_cast<int>(max(static_cast<int64_t>(v.pos0) - p.window + 1, int64_t(0))) : 0;
  v.first_page = min(from, last) / kPage;
  const int sink_pages = min((p.sinks + int64_t(kPage - 1)) / kPage, static_cast<int64_t>(v.first_page));
  v.sink_tiles = sink_pages;
  v.tiles = v.sink_tiles + last / kPage - v.first_page + 1;
  return v;
}

// Rows i (tokens) of the unit that see position j: i in [lo, hi).
__device__ __forceinline__ void rows_that_see(const AttentionParams& p, const SeqView& v, int j, bool page_ok, int& lo, int& hi) {
  const int64_t d = static_cast<int64_t>(j) - v.pos0;
  lo = static_cast<int>(min(max(d, int64_t(0)), int64_t(v.n)));
  hi = v.n;
  if (p.window > 0 && j >= p.sinks) hi = static_cast<int>(min(max(d + p.window, int64_t(0)), int64_t(v.n)));
  if (!page_ok || j >= v.len) hi = 0;
}

}  // namespace tg
