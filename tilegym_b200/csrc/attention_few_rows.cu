// Attention over the paged e4m3 cache for few rows: R = (new tokens of a sequence) * (query heads of a cache head) <= 32.
//
// The cache's bytes are read once and are nearly all of the work, so the kernel is built to keep copies in flight, and the
// cached bytes ARE the tensor core's operands: no conversion, no transposition.
//
//   S^T [128 tokens, R]  = K [128, dim] . Q^T           kind::f8f6f4, q = q1 + q2 (+ q3) in e4m3, summed by the accumulator
//   p = 2^(S * scale * log2 e + log2 v_scale - ref)     thread = token; v_scale of the page rides in the exponent
//   O^T [dim, R]        += V^T [dim, 128] . P           p = p1 + p2 + p3 (+ p4) in e5m2, beside V's e4m3
//
// The two factors that are not in the cache are split into 8-bit terms, each holding what the one before left, which stand
// side by side as rows of the operand, so a page is read once for all of them; their columns of S^T and O^T are joined by the
// softmax and at the end.  q: e4m3, each term kept 16 times larger than the one before; two hold a bf16 exactly, three (f16) to
// 2^-12.  p: rounded to f16, then cut into e5m2, which is f16's upper byte, 8 times larger each; three terms (bf16) hold it
// to 2^-9, four (f16) hold the f16 whole.  p needs the range of f16, not of e4m3: where one token has most of a row's weight,
// a long cache shares the rest among weights 2^-20 of the largest and below, and the sum counts them whatever becomes of them
// in the product.  A row's largest p is kept between 2^9 and 2^14, so the terms keep their relative rounding down to 2^-23
// of it and end at 2^-32 (2^-34 with four).
// `ref` is a running maximum of the exponent that is only moved when a p would pass 2^14 (2^5 of headroom), which rescales O^T
// in TMEM.  Keeping v_scale in the exponent keeps p at one magnitude whatever the pages' scales are.
//
// Work: the pages that the units (sequence, cache head) see are numbered through, each unit kUnitCost numbers in front of
// them for what it costs to begin and end one, and every block takes an equal range of the numbers, wherever that begins
// and ends: no batch is too ragged.  A block that ends inside a unit leaves a partial result and
// a record; the joining kernel adds the parts of such a unit in block order, so results do not depend on timing.
// Warp 0 copies pages (TMA, a ring of page pairs), warps 1 and 2 issue the two products, warps 3-6 do the softmax.  Where the shared
// memory holds one block per SM only, four more warps share it: the two groups take pages in turn, each with references,
// sums and an O^T of its own, which are joined when the unit ends (the softmax of 32 rows takes longer than copying the page).
//
// Bound: HBM up to 16 rows, the chain of the softmax from there.  Measured (8 cache heads of 128, bf16): 64 sequences of up to
// 16000 tokens with 4 rows 173 us (1.1 GB, 0.97 of the copy bandwidth); 37 sequences of 8000 with 32 rows 160 us (0.58); one
// sequence of 2001 tokens 12.7 us, of 32000 25 us.  Of 64 sequences of up to 8000 tokens (f16), equal shares counted in pages alone
// took 164 us, with what units cost counted in 103.
#include <cstdio>

#include "tg_attention.cuh"

namespace tg {
namespace {

constexpr float kNominal = 9.f, kLimit = 14.f;  // p is kept times 2^9 and may reach 2^14 (e5m2 ends at 2^15.8) before ref moves
constexpr float kUnset = -1e30f;  // the reference of a row that has not seen a token yet

template <typename T>
constexpr int kTermsOf = std::is_same<T, __half>::value ? 3 : 2;  // of q; p has one more

template <int DIM, int N, int TERMS>
struct Shape {
  static constexpr int kTile = DIM * kPage;  // bytes of a key or value page
  static constexpr int kPTerms = TERMS + 1;
  static constexpr int kP = (kPTerms * N + 31) / 32 * 32 * kPage;  // planes of [token][32 columns]
  static constexpr int kQ = TERMS * N * DIM;
  // two blocks share an SM where each still has a ring of three page pairs
  static constexpr int kBlocksPerSm = N == 16 && !(TERMS == 3 && DIM == 128) ? 2 : 1;
  static constexpr int kGroups = kBlocksPerSm == 2 ? 1 : 2;  // of four softmax warps
  static constexpr int kThreads = 96 + 128 * kGroups;
  // Each group has a buffer of P.  One group with two buffers would not leave room for three page pairs, and gains nothing by
  // them: the product of the page before is done long before this page's exponentials are.
  static constexpr int kPAll = kGroups * kP;
  // A unit's queries, first references and result take about 8000 clocks; a page 2000 (one group, two blocks to share the
  // SM) or 1100.
  static constexpr int kUnitCost = kGroups == 1 ? 4 : 6;
  // barriers and notes; row factors; references; maxima and sums; rows that see a NaN
  static constexpr int kRowmul = 1024, kRef = kRowmul + N * 4, kWmax = kRef + kGroups * 2 * N * 4, kNan = kWmax + kGroups * 2 * 4 * N * 4;
  static constexpr int kMisc = kNan + (kGroups == 2 ? 2 * 128 * 4 : 0);
  // dim 64: the value operand is read as 128 rows, 64 of them whatever follows the page
  static constexpr int kBudget = (kBlocksPerSm == 2 ? 113 : 226) * 1024 - 1024 - kPAll - kQ - kMisc;
  static constexpr int kStages = kBudget / (2 * kTile) > 8 ? 8 : kBudget / (2 * kTile);
  static constexpr int kSmem = 1024 + kStages * 2 * kTile + kPAll + kQ + kMisc;
  static constexpr int kSCols = TERMS * N;  // q's terms have columns of their own in S^T
  static constexpr int kOCols = kPTerms * N;   // and p's in O^T
  static constexpr int kTmemUsed = 2 * kSCols + kGroups * kOCols;  // S^T twice and each group's O^T by term
  static constexpr int kTmem = kTmemUsed <= 128 ? 128 : kTmemUsed <= 256 ? 256 : 512;
  static_assert(kStages >= 3, "the ring is too short to hide the latency of a page");
  static_assert(kPAll + kQ >= 8192, "the value operand of dim 64 reads 8 KB behind its page");
};

struct TileInfo {
  float ks, lv, inv_vs;
  int base;  // position of the page's first token; -1: no such page
};

// The operand P [columns][tokens] with the columns together: planes of 32 columns (32 bytes per token, tokens one after the
// other, the two halves changing places every four tokens: the 32-byte swizzle), 4 KB from one plane to the next and 256 bytes
// from one group of eight tokens to the next.  A thread, which has a token, writes eight columns at once; with the tokens
// together every byte was a store of its own (32 rows, f16, dim 64, 37 sequences of 8000, with three terms: 163 us, 190 that way).
// B's format is e5m2 (idesc bits 10-12), its columns lie together (bit 16).
__device__ __forceinline__ uint64_t columns_desc(uint32_t smem_addr) {
  return static_cast<uint64_t>((smem_addr >> 4) & 0x3FFFu) | (static_cast<uint64_t>((32 * kPage) >> 4) << 16) | (static_cast<uint64_t>(256u >> 4) << 32) |
         (1ull << 46) | (6ull << 61);
}

// A bounded wait whose outcome is the same for the whole warp, which is converged behind it.
template <bool kHint = false>
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile uint32_t* abort_flag) {
  return __all_sync(0xffffffffu, mbar_wait<kHint>(bar, parity, abort_flag));
}

// Eight values as sums of TERMS times eight e5m2 values, each term kPStep times larger than it is beside the one before.  e5m2 is
// the upper byte of f16 and holds three significant bits: cutting a positive f16 there leaves less than a quarter of its leading
// bit, exactly.  The last term is rounded to even; four hold all eleven bits, subnormal ones too.
constexpr float kPStep = 8.f;
template <int TERMS>
__device__ __forceinline__ void split_e5m2(const float (&p)[8], uint32_t (&term)[TERMS][2]) {
  uint32_t h[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) h[j] = pack_pair<__half>(p[2 * j], p[2 * j + 1]);
#pragma unroll
  for (int x = 0; x < TERMS; ++x) {
    if (x + 1 == TERMS) {
#pragma unroll
      for (int j = 0; j < 4; ++j) h[j] += 0x007f007fu + ((h[j] >> 8) & 0x00010001u);
    }
    term[x][0] = __byte_perm(h[0], h[1], 0x7531);
    term[x][1] = __byte_perm(h[2], h[3], 0x7531);
    if (x + 1 == TERMS) break;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t cut = h[j] & 0xff00ff00u;
      const __half2 rest = __hmul2(__hsub2(*reinterpret_cast<const __half2*>(&h[j]), *reinterpret_cast<const __half2*>(&cut)), __float2half2_rn(kPStep));
      h[j] = *reinterpret_cast<const uint32_t*>(&rest);
    }
  }
}

__device__ __forceinline__ void load8(const float* src, float (&v)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(src), b = *reinterpret_cast<const float4*>(src + 4);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}

// Softmax warps meet at a hardware barrier (`count` threads); true if any thread says so.  Nobody waits alone here: whatever a
// warp found, it comes.
__device__ __forceinline__ bool softmax_vote(uint32_t barrier, uint32_t count, bool mine) {
  uint32_t any;
  asm volatile(
      "{\n\t"
      ".reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, %2, %3, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t"
      "}"
      : "=r"(any)
      : "r"(static_cast<uint32_t>(mine)), "r"(barrier), "r"(count)
      : "memory");
  return any != 0;
}

// The units are numbered sequence by sequence, the cache heads of a sequence next to one another.
struct Cursor {
  int b, h;
  SeqView v;
};
__device__ __forceinline__ bool next_unit(const AttentionParams& p, Cursor& c) {
  if (++c.h < p.c.heads) return true;
  c.h = 0;
  do {
    if (++c.b >= p.c.seqs) return false;
    c.v = view_sequence(p, c.b, 0, p.max_q_len);
  } while (c.v.tiles == 0);
  return true;
}

// One element's row of a value page (128 tokens) of which not every row sees every token.  Values that nobody sees are
// whatever memory held, NaN among it, and 0 * NaN is NaN: they become zeros.  A NaN that some rows see is kept from the
// product, which would give it to all, and noted for those rows.
__device__ __noinline__ void clean_values(const AttentionParams& p, const SeqView& v, int base, uint8_t* row, int d, uint32_t& nan_rows) {
  // tokens of the page that some row sees: t < hi and (t >= lo or t < sink)
  const int hi = base >= 0 ? min(max(min(v.len, v.pos0 + v.n) - base, 0), kPage) : 0;
  const int lo = p.window > 0 ? static_cast<int>(min(max(static_cast<int64_t>(v.pos0) - p.window + 1 - base, int64_t(0)), int64_t(kPage))) : 0;
  const int sink = min(max(p.sinks - max(base, 0), 0), kPage);
#pragma unroll 2
  for (int c = 0; c < kPage / 16; ++c) {
    uint4* at = reinterpret_cast<uint4*>(row + ((c ^ (d & 7)) << 4));
    const int t = c * 16;
    if (t >= hi || (t >= sink && t + 16 <= lo)) {
      *at = make_uint4(0, 0, 0, 0);
      continue;
    }
    const bool all = t + 16 <= hi && (t >= lo || t + 16 <= sink);
    const uint4 w = *at;
    uint32_t ww[4] = {w.x, w.y, w.z, w.w};
    if (!all) {
#pragma unroll
      for (int x = 0; x < 16; ++x)
        if (!(t + x < hi && (t + x >= lo || t + x < sink))) ww[x >> 2] &= ~(255u << (8 * (x & 3)));
    }
    uint32_t nan = 0;
#pragma unroll
    for (int x = 0; x < 4; ++x) nan |= ((ww[x] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
    if (nan) {
#pragma unroll 1
      for (int x = 0; x < 16; ++x) {
        const uint32_t word = x < 8 ? (x < 4 ? ww[0] : ww[1]) : (x < 12 ? ww[2] : ww[3]);
        if (((word >> (8 * (x & 3))) & 127u) != 127u) continue;
        int a, z;
        rows_that_see(p, v, base + t + x, true, a, z);
        a *= p.group;
        z *= p.group;
        if (a < z) nan_rows |= (z >= 32 ? ~0u : (1u << z) - 1) & ~((1u << a) - 1);
        const uint32_t keep = ~(255u << (8 * (x & 3)));
        if (x < 4) ww[0] &= keep;
        else if (x < 8) ww[1] &= keep;
        else if (x < 12) ww[2] &= keep;
        else ww[3] &= keep;
      }
    }
    if (nan || !all) *at = make_uint4(ww[0], ww[1], ww[2], ww[3]);
  }
}

template <typename T, int DIM, int N>
__global__ void __launch_bounds__((Shape<DIM, N, kTermsOf<T>>::kThreads), (Shape<DIM, N, kTermsOf<T>>::kBlocksPerSm))
    tg_attention_few_rows_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ AttentionParams p) {
  constexpr int kTerms = kTermsOf<T>;
  using Sh = Shape<DIM, N, kTerms>;
  constexpr int kStages = Sh::kStages, kGroups = Sh::kGroups, kThreads = Sh::kThreads, kPTerms = Sh::kPTerms, kOCols = Sh::kOCols;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* p_smem = smem + kStages * 2 * Sh::kTile;
  uint8_t* q_smem = p_smem + Sh::kPAll;
  uint8_t* misc = q_smem + Sh::kQ;
  // misc: barriers, tile notes, row factors, exchanged maxima
  uint64_t* bars = reinterpret_cast<uint64_t*>(misc);
  TileInfo* info = reinterpret_cast<TileInfo*>(misc + 512);
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(misc + 512 + 8 * sizeof(TileInfo));
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(misc + 512 + 8 * sizeof(TileInfo) + 16);
  int64_t* sched = reinterpret_cast<int64_t*>(misc + 512 + 8 * sizeof(TileInfo) + 32);  // 0 tiles in front, 1 sequence, 2.. warp sums
  float* rowmul = reinterpret_cast<float*>(misc + Sh::kRowmul);

  const uint32_t bar0 = smem_u32(bars);
  const uint32_t b_full = bar0, b_empty = bar0 + 8 * kStages, b_sfull = b_empty + 8 * kStages, b_sempty = b_sfull + 16,
                 b_pready = b_sempty + 16, b_pvdone = b_pready + 16, b_qready = b_pvdone + 16;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (warp == 0) {
    if (elect_one()) {
      prefetch_tmap(&tmK);
      prefetch_tmap(&tmV);
    }
    if (lane == 0) {
      for (int i = 0; i < kStages; ++i) {
        mbar_init(b_full + 8 * i, 1);
        mbar_init(b_empty + 8 * i, 1);
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(b_sfull + 8 * i, 1);
        mbar_init(b_sempty + 8 * i, 4);
        mbar_init(b_pready + 8 * i, 4);
        mbar_init(b_pvdone + 8 * i, 1);
      }
      mbar_init(b_qready, 4 * kGroups);
      init_abort_flag(abort_flag, p.wait_limit_us);
      fence_mbar_init();
    }
  } else if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), Sh::kTmem);
    tmem_relinquish();
  }
  griddep_wait();
  griddep_launch_dependents();

  // ---- this block's range of pages
  int64_t total, begin = 0, end = 0, blocks, front = 0;
  Cursor cur;
  cur.b = -1;
  cur.v = SeqView{};
  auto numbers = [](const SeqView& v) { return v.tiles > 0 ? v.tiles + Sh::kUnitCost : 0; };
  auto divide = [&]() {
    total *= p.c.heads;
    blocks = min(static_cast<int64_t>(gridDim.x), total);  // the others have nothing to do
    if (blockIdx.x < blocks) {
      begin = total * blockIdx.x / blocks;
      end = total * (blockIdx.x + 1) / blocks;
    }
  };
  if (p.c.seqs <= 32) {
    // a lane per sequence, every warp for itself: no barrier in the way of a small batch
    SeqView v = {};
    if (lane < p.c.seqs) v = view_sequence(p, lane, 0, p.max_q_len);
    const int n = numbers(v);
    int64_t incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    total = __shfl_sync(0xffffffffu, incl, 31);
    divide();
    if (begin < end) {
      const int64_t target = begin / p.c.heads;
      const uint32_t hit = __ballot_sync(0xffffffffu, n > 0 && incl - n <= target && target < incl);
      cur.b = __ffs(hit) - 1;
      front = __shfl_sync(0xffffffffu, incl - n, cur.b);
      cur.v.lo = __shfl_sync(0xffffffffu, v.lo, cur.b);
      cur.v.n = __shfl_sync(0xffffffffu, v.n, cur.b);
      cur.v.len = __shfl_sync(0xffffffffu, v.len, cur.b);
      cur.v.pos0 = __shfl_sync(0xffffffffu, v.pos0, cur.b);
      cur.v.tiles = __shfl_sync(0xffffffffu, v.tiles, cur.b);
      cur.v.sink_tiles = __shfl_sync(0xffffffffu, v.sink_tiles, cur.b);
      cur.v.first_page = __shfl_sync(0xffffffffu, v.first_page, cur.b);
    }
  } else {
    const int mine = static_cast<int>(threadIdx.x) < p.c.seqs ? numbers(view_sequence(p, threadIdx.x, 0, p.max_q_len)) : 0;
    int64_t sum = mine;
    for (int b = threadIdx.x + kThreads; b < p.c.seqs; b += kThreads) sum += numbers(view_sequence(p, b, 0, p.max_q_len));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) sched[2 + warp] = sum;
    if (threadIdx.x == 0) sched[1] = -1;
    __syncthreads();
    total = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) total += sched[2 + w];
    divide();
    // the sequence in which it begins: prefix sums, as far as needed
    const int64_t target = begin / p.c.heads;
    int64_t before = 0;
    for (int base = 0; base < p.c.seqs && begin < end; base += kThreads) {
      const int b = base + threadIdx.x;
      const int n = base == 0 ? mine : b < p.c.seqs ? numbers(view_sequence(p, b, 0, p.max_q_len)) : 0;
      int64_t incl = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
      }
      __syncthreads();
      if (lane == 31) sched[2 + warp] = incl;
      __syncthreads();
      int64_t off = before, all = before;
#pragma unroll
      for (int w = 0; w < kThreads / 32; ++w) {
        if (w < warp) off += sched[2 + w];
        all += sched[2 + w];
      }
      if (n > 0 && off + incl - n <= target && target < off + incl) {
        sched[0] = off + incl - n;
        sched[1] = b;
      }
      before = all;
      if (before > target) break;  // the same for every thread
    }
    __syncthreads();
    cur.b = begin < end ? static_cast<int>(sched[1]) : -1;
    if (cur.b >= 0) {
      front = sched[0];
      cur.v = view_sequence(p, cur.b, 0, p.max_q_len);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  int from = 0;  // number within the unit at which this block's part begins
  const bool work = begin < end && cur.b >= 0;
  if (work) {
    const int64_t rem = begin - front * p.c.heads;
    const int each = numbers(cur.v);
    cur.h = rem <= 0xffffffffll ? static_cast<int>(static_cast<uint32_t>(rem) / static_cast<uint32_t>(each)) : static_cast<int>(rem / each);
    from = static_cast<int>(rem - static_cast<int64_t>(cur.h) * each);
  } else if (threadIdx.x == 0) {
    p.record[blockIdx.x] = make_int4(-1, 0, 0, 0);
  }
  // this block's pages [t0, t1) of the current unit; false: the range ended in front of the unit's first page
  int t0 = 0, t1 = 0;
  int64_t left = work ? end - begin : 0;
  auto take = [&]() {
    const int to = static_cast<int>(min(static_cast<int64_t>(numbers(cur.v)), from + left));
    left -= to - from;
    t0 = max(from - Sh::kUnitCost, 0);
    t1 = max(to - Sh::kUnitCost, 0);
    from = 0;
    return t1 > t0;
  };
  bool ok = true;
  int site = 0;

  if (warp == 0) {
    // ------------------------------------------------------------------------------------------ copies
    const uint64_t policy = policy_evict_first();
    const int rows_k = p.c.pages * p.c.heads * kPage, rows_v = p.c.pages * p.c.heads * DIM;
    int it = 0;
    while (left > 0 && ok) {
      if (!take()) break;
      for (int base = t0; base < t1 && ok; base += 32) {
        // 32 pages at a time: numbers first, so that copies start before the scales are here
        const int t = base + lane;
        const int page = t < t1 ? cur.v.page_of(t) : p.c.max_pages;
        int phys = page < p.c.max_pages ? p.c.table[cur.b * p.c.table_pitch + page] : -1;
        if (phys < 0 || phys >= p.c.pages) phys = -1;
        const int64_t block = static_cast<int64_t>(phys) * p.c.heads + cur.h;
        float ks = 0.f, vs = 1.f;
        if (phys >= 0) {
          ks = p.c.ks[block];
          vs = p.c.vs[block];
        }
        for (int i = 0; i < min(32, t1 - base); ++i, ++it) {
          const int stage = it % kStages, round = it / kStages;
          if (!warp_wait<true>(b_empty + 8 * stage, (round & 1) ^ 1, abort_flag)) {
            ok = false;
            site = 1;
            break;
          }
          const int ph = __shfl_sync(0xffffffffu, phys, i);
          // a page that is not there: a box behind the end of the cache, which reads as zeros
          const int yk = ph >= 0 ? (ph * p.c.heads + cur.h) * kPage : rows_k;
          const int yv = ph >= 0 ? (ph * p.c.heads + cur.h) * DIM : rows_v;
          const uint32_t dst = smem_u32(smem + stage * 2 * Sh::kTile);
          if (elect_one()) {
            tma_load_2d_hint(dst, &tmK, b_full + 8 * stage, 0, yk, policy);
            tma_load_2d_hint(dst + Sh::kTile, &tmV, b_full + 8 * stage, 0, yv, policy);
          }
          __syncwarp();
          const float k1 = __shfl_sync(0xffffffffu, ks, i), v1 = __shfl_sync(0xffffffffu, vs, i);
          if (elect_one()) {
            info[stage] = TileInfo{k1, log2f(v1), 1.0f / v1, ph >= 0 ? cur.v.page_of(base + i) * kPage : -1};
            mbar_arrive_expect_tx(b_full + 8 * stage, 2 * Sh::kTile);
          }
          __syncwarp();
        }
      }
      if (left > 0 && !next_unit(p, cur)) break;
    }
    if (!ok) {
      if (lane == 0) *p.status = kRoleProducer * 1000 + site;
      // copies still in flight land before the block leaves (a bounded number of parked tries each)
      for (int i = max(it - kStages, 0); i < it; ++i)
        for (int tries = 0; tries < 1000 && !mbar_try_wait(b_full + 8 * (i % kStages), (i / kStages) & 1); ++tries) {
        }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------------------------------ scores
    constexpr uint32_t idesc = make_idesc_e4m3_f32(128, Sh::kSCols);
    const uint32_t q_addr = smem_u32(q_smem);
    int it = 0, unit = 0;
    while (left > 0 && ok) {
      if (!take()) break;
      if (!warp_wait(b_qready, unit & 1, abort_flag)) {
        ok = false;
        site = 1;
        break;
      }
      ++unit;
      for (int t = t0; t < t1; ++t, ++it) {
        const int stage = it % kStages, buf = it & 1;
        if (!warp_wait(b_full + 8 * stage, (it / kStages) & 1, abort_flag) ||
            !warp_wait(b_sempty + 8 * buf, ((it >> 1) & 1) ^ 1, abort_flag)) {
          ok = false;
          site = 2;
          break;
        }
        tc_fence_after();
        if (elect_one()) {
          const uint64_t a = rows_desc<DIM>(smem_u32(smem + stage * 2 * Sh::kTile));
          const uint64_t b = rows_desc<DIM>(q_addr);
#pragma unroll
          for (int k = 0; k < DIM / 32; ++k) mma_f8f6f4(tmem + buf * Sh::kSCols, a + 2 * k, b + 2 * k, idesc, k > 0);
          tc_commit(b_sfull + 8 * buf);
        }
        __syncwarp();
      }
      if (left > 0 && !next_unit(p, cur)) break;
    }
    if (!ok && lane == 0) *p.status = kRoleMma * 1000 + site;
  } else if (warp == 2) {
    // ------------------------------------------------------------------------------------------ values
    constexpr uint32_t idesc = make_idesc_e4m3_f32(128, kOCols) | (1u << 10) | (1u << 16);
    const uint32_t p_addr = smem_u32(p_smem);
    int it = 0;
    while (left > 0 && ok) {
      if (!take()) break;
      for (int t = t0; t < t1; ++t, ++it) {
        const int stage = it % kStages, buf = it & 1;
        if (!warp_wait(b_pready + 8 * buf, (it >> 1) & 1, abort_flag)) {
          ok = false;
          site = 3;
          break;
        }
        tc_fence_after();
        if (elect_one()) {
          const uint64_t a = make_kmajor_sw128_desc(smem_u32(smem + stage * 2 * Sh::kTile + Sh::kTile));
          const uint64_t b = columns_desc(p_addr + (kGroups == 2 ? buf * Sh::kP : 0));
          const bool more = t - t0 >= kGroups;  // the group has an O^T of this unit already
#pragma unroll
          for (int k = 0; k < kPage / 32; ++k)
            mma_f8f6f4(tmem + 2 * Sh::kSCols + (kGroups == 2 ? buf * kOCols : 0), a + 2 * k, b + 64 * k, idesc, more || k > 0);
          // the softmax has had S^T, so both of the stage's pages are done with
          tc_commit(b_empty + 8 * stage);
          tc_commit(b_pvdone + 8 * buf);
        }
        __syncwarp();
      }
      if (left > 0 && !next_unit(p, cur)) break;
    }
    if (!ok && lane == 0) *p.status = kRoleMma * 1000 + site;
  } else {
    // ------------------------------------------------------------------------------------------ softmax
    // A wait that gives up is remembered, not acted on: the warps leave together at their next vote, a group's own (which
    // ends its pages) or the one of all.
    const int quarter = warp & 3, token = quarter * 32 + lane, at = (warp - 3) * 32 + lane, group = kGroups == 2 ? at >> 7 : 0;
    const int st = at & 127;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t t_all = tmem + 2 * Sh::kSCols + lane_off, t_o = t_all + group * kOCols;
    float* refs = reinterpret_cast<float*>(misc + Sh::kRef);          // [group][copy][N]
    float* ref = refs + group * 2 * N;
    float* maxima = reinterpret_cast<float*>(misc + Sh::kWmax);       // [group][copy][4][N]: the warps' maxima, or sums, by row
    float* wmax = maxima + group * 8 * N;
    int2* side_notes = reinterpret_cast<int2*>(misc + 960);           // [group]: which copies hold its sums and references
    uint32_t* nan_notes = reinterpret_cast<uint32_t*>(misc + Sh::kNan);  // [group][element of the head]
    auto vote = [&](bool mine) { return softmax_vote(1 + group, 128, mine); };
    auto vote_all = [&](bool mine) { return softmax_vote(kGroups == 2 ? 3 : 1, 128 * kGroups, mine); };
    int it = 0, turn = 0;
    int64_t number_at = begin - from;  // of the current unit
    int4 rec = make_int4(-1, 0, 0, 0);
    float l[N];
    int side = 0;  // which of the two copies of the references holds
    auto wait = [&](uint32_t bar, uint32_t parity, int where) {
      if (!warp_wait(bar, parity, abort_flag) && ok) {
        ok = false;
        site = where;
      }
    };
    while (left > 0) {
      if (!take()) break;
      const SeqView v = cur.v;
      const int rows = v.n * p.group;
      // ---- queries: eight elements per thread, split into e4m3 terms under a power-of-two scale of their row
      {
        constexpr int kLanes = DIM / 8, kRows = 128 * kGroups / kLanes, kPasses = (N + kRows - 1) / kRows, kBatch = kPasses < 4 ? kPasses : 4;
        const int e = (at % kLanes) * 8;
#pragma unroll 1
        for (int r0 = 0; r0 < rows; r0 += kRows * kBatch) {
          uint4 w[kBatch];
#pragma unroll
          for (int k = 0; k < kBatch; ++k) {
            const int r = r0 + k * kRows + at / kLanes, i = r / p.group;
            w[k] = make_uint4(0, 0, 0, 0);
            if (r < rows)
              w[k] = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + (v.lo + i) * p.q_tok + (cur.h * p.group + r - i * p.group) * p.q_head + e);
          }
#pragma unroll
          for (int k = 0; k < kBatch; ++k) {
            const int r = r0 + k * kRows + at / kLanes;
            const uint32_t ww[4] = {w[k].x, w[k].y, w[k].z, w[k].w};
            float f[8];
            uint32_t top = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float2 u = unpack_pair<T>(ww[j]);
              f[2 * j] = u.x;
              f[2 * j + 1] = u.y;
              top = max(top, max(__float_as_uint(u.x) & 0x7fffffffu, __float_as_uint(u.y) & 0x7fffffffu));
            }
#pragma unroll
            for (int o = kLanes / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
            const float sc = cache_scale(__uint_as_float(top)), inv = pow2_reciprocal(sc);
            uint32_t out[kTerms][2];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              uint32_t term[kTerms];
              split_e4m3<kTerms>(f[2 * j] * inv, f[2 * j + 1] * inv, kTermStep, term);
#pragma unroll
              for (int x = 0; x < kTerms; ++x) out[x][j >> 1] = (j & 1) ? out[x][j >> 1] | (term[x] << 16) : term[x];
            }
            if (r < N) {
#pragma unroll
              for (int x = 0; x < kTerms; ++x)
                *reinterpret_cast<uint2*>(q_smem + x * N * DIM + swizzled<DIM>(r, e)) = make_uint2(out[x][0], out[x][1]);
              // a row that holds an infinity or NaN has no answer
              if (e == 0) rowmul[r] = top >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : sc * p.scale * 1.4426950408889634f;
            }
          }
        }
        // rows that fill up a group of eight: exponents of minus infinity.  The copy that nobody can still be reading.
        side ^= 1;
        if (st < N) ref[side * N + st] = st < rows ? kUnset : INFINITY;
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(b_qready);
        if (vote_all(!ok)) break;
      }
#pragma unroll
      for (int r = 0; r < N; ++r) l[r] = 0.f;
      uint32_t nan_rows = 0;  // rows that see a NaN in element `token` of a value
      // positions that every row sees: [all_lo, all_hi), and the first tokens
      const int all_hi = min(v.len, v.pos0 + 1);
      const int all_lo = p.window > 0 ? static_cast<int>(max(static_cast<int64_t>(v.pos0) + v.n - p.window, int64_t(0))) : 0;
      int mine = 0;  // pages of this unit that this group has done
      for (int t = t0; t < t1; ++t, ++it) {
        const int stage = it % kStages, buf = it & 1;
        if (kGroups == 2 && buf != group) continue;
        wait(b_full + 8 * stage, (it / kStages) & 1, 1);
        const TileInfo ti = info[stage];
        const bool whole = ti.base >= 0 && ti.base + kPage <= all_hi && (ti.base >= all_lo || ti.base + kPage <= p.sinks);
        int see_lo = 0, see_hi = N;
        if (!whole) {
          rows_that_see(p, v, ti.base + token, ti.base >= 0, see_lo, see_hi);
          see_lo *= p.group;
          see_hi *= p.group;
          if (token < DIM) clean_values(p, v, ti.base, smem + stage * 2 * Sh::kTile + Sh::kTile + token * kPage, token, nan_rows);
        }
        wait(b_sfull + 8 * buf, (it >> 1) & 1, 2);
        tc_fence_after();
        const uint32_t t_s = tmem + buf * Sh::kSCols + lane_off;
        // ---- exponents: z = S * (row's factor * page's scale) + log2 v_scale - ref + kNominal, eight rows at a time
        float z[N];
        const float shift = ti.lv + kNominal;
        auto exponents = [&](bool with_ref) {
#pragma unroll
          for (int c = 0; c < N; c += 16) {
            if (c >= rows) break;
            uint32_t part[kTerms][16];
#pragma unroll
            for (int x = 0; x < kTerms; ++x) tmem_ld_32x16(t_s + x * N + c, part[x]);
            tmem_ld_wait();
            float s[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              s[j] = __uint_as_float(part[kTerms - 1][j]);
#pragma unroll
              for (int x = kTerms - 2; x >= 0; --x) s[j] = fmaf(s[j], 1.f / kTermStep, __uint_as_float(part[x][j]));
            }
#pragma unroll
            for (int g = 0; g < 16; g += 8) {
              if (c + g >= rows) break;
              float m[8], r[8];
              load8(rowmul + c + g, m);
              load8(ref + side * N + c + g, r);
#pragma unroll
              for (int j = 0; j < 8; ++j) z[c + g + j] = fmaf(s[g + j], m[j] * ti.ks, with_ref ? shift - r[j] : shift);
            }
          }
          if (!whole) {
#pragma unroll
            for (int r = 0; r < N; ++r)
              if (r < see_lo || r >= see_hi) z[r] = -INFINITY;
          }
        };
        bool move = mine == 0;
        if (!move) {
          exponents(true);
          float over = -INFINITY;
#pragma unroll
          for (int g = 0; g < N; g += 8) {
            if (g >= rows) break;
            over = fmaxf(over, fmaxf(fmaxf(fmaxf(z[g], z[g + 1]), fmaxf(z[g + 2], z[g + 3])), fmaxf(fmaxf(z[g + 4], z[g + 5]), fmaxf(z[g + 6], z[g + 7]))));
          }
          move = vote(over > kLimit || !ok);
        }
        if (move) {
          // ---- some row's exponent has outgrown its reference (or has none yet): every row's maximum, and a new reference
          // where it is needed; the sums and O^T go along
          exponents(false);
          float* wm = wmax + (turn & 1) * 4 * N;
          ++turn;
#pragma unroll
          for (int g = 0; g < N; g += 8) {
            if (g >= rows) break;
            float m[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) m[j] = redux_max(z[g + j]);
            if (lane == 0) {
              *reinterpret_cast<float4*>(wm + quarter * N + g) = make_float4(m[0], m[1], m[2], m[3]);
              *reinterpret_cast<float4*>(wm + quarter * N + g + 4) = make_float4(m[4], m[5], m[6], m[7]);
            }
          }
          const int last = it - kGroups;  // this group's page before
          if (mine > 0) wait(b_pvdone + 8 * (last & 1), (last >> 1) & 1, 3);
          if (vote(!ok)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const float* old = ref + side * N;
          float* now = ref + (side ^ 1) * N;
#pragma unroll
          for (int g = 0; g < N; g += 8) {
            if (g >= rows) break;
            float top[8], was[8], f[8];
            load8(wm + g, top);
#pragma unroll
            for (int q = 1; q < 4; ++q) {
              float w[8];
              load8(wm + q * N + g, w);
#pragma unroll
              for (int j = 0; j < 8; ++j) top[j] = fmaxf(top[j], w[j]);
            }
            load8(old + g, was);
            bool any = false;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float m = top[j] - kNominal;
              const bool go = m > was[j] + (kLimit - kNominal) || was[j] == kUnset;
              const float r = go ? fmaxf(m, kUnset) : was[j];
              any = any || go;
              f[j] = exp2_approx(was[j] - r);
              l[g + j] *= f[j];
              z[g + j] -= r;
              top[j] = r;
            }
            if (st == 0) {
              *reinterpret_cast<float4*>(now + g) = make_float4(top[0], top[1], top[2], top[3]);
              *reinterpret_cast<float4*>(now + g + 4) = make_float4(top[4], top[5], top[6], top[7]);
            }
            if (mine > 0 && any) {
              uint32_t o[kPTerms][8];
#pragma unroll
              for (int x = 0; x < kPTerms; ++x) tmem_ld_32x8(t_o + x * N + g, o[x]);
              tmem_ld_wait();
#pragma unroll
              for (int x = 0; x < kPTerms; ++x) {
#pragma unroll
                for (int j = 0; j < 8; ++j) o[x][j] = __float_as_uint(__uint_as_float(o[x][j]) * f[j]);
                tmem_st_32x8(t_o + x * N + g, o[x]);
              }
            }
          }
          if (mine > 0) tmem_st_wait();
          side ^= 1;
          if (vote(!ok)) {
            ok = false;
            break;
          }
        }
        ++mine;
        // ---- P; its buffer is free once the group's product before has read it
        wait(b_pvdone + 8 * ((it - kGroups) & 1), ((it - kGroups) >> 1) & 1, 5);
        const uint32_t pb = smem_u32(p_smem) + group * Sh::kP + token * 32, flip = (token & 4) << 2;
#pragma unroll
        for (int g = 0; g < N; g += 8) {
          if (g >= rows) break;
          float e[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            e[j] = exp2_approx(z[g + j]);
            // the sums take p as it is: a page whose values are tiny beside the others' still counts in full
            l[g + j] = fmaf(e[j], ti.inv_vs, l[g + j]);
          }
          uint32_t word[kPTerms][2];
          split_e5m2<kPTerms>(e, word);
#pragma unroll
          for (int x = 0; x < kPTerms; ++x) {
            const int col = x * N + g;
            asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(pb + (col >> 5) * (32 * kPage) + ((col & 16) ^ flip) + (col & 8)), "r"(word[x][0]), "r"(word[x][1]) : "memory");
          }
        }
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(b_sempty + 8 * buf);
          mbar_arrive(b_pready + 8 * buf);
        }
      }
      // ---- the unit's (or this block's part of its) result: thread = element of the head
      // the groups' copies: the other one has to know where to look
      if (kGroups == 2 && st == 0) side_notes[group] = make_int2(turn & 1, side);
      float* sums = wmax + (turn & 1) * 4 * N;
      ++turn;
#pragma unroll
      for (int g = 0; g < N; g += 8) {
        if (g >= rows) break;
        // eight sums over 32 lanes: each step halves the values a lane still carries, lane i ends with row i mod 8
        float a[4], b2[2], c;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float give = (lane & 4) ? l[g + j] : l[g + j + 4], keep = (lane & 4) ? l[g + j + 4] : l[g + j];
          a[j] = keep + __shfl_xor_sync(0xffffffffu, give, 4);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float give = (lane & 2) ? a[j] : a[j + 2], keep = (lane & 2) ? a[j + 2] : a[j];
          b2[j] = keep + __shfl_xor_sync(0xffffffffu, give, 2);
        }
        {
          const float give = (lane & 1) ? b2[0] : b2[1], keep = (lane & 1) ? b2[1] : b2[0];
          c = keep + __shfl_xor_sync(0xffffffffu, give, 1);
        }
        c += __shfl_xor_sync(0xffffffffu, c, 8);
        c += __shfl_xor_sync(0xffffffffu, c, 16);
        if (lane < 8) sums[quarter * N + g + lane] = c;
      }
      if (mine > 0) {
        const int last = kGroups == 2 && ((it - 1) & 1) != group ? it - 2 : it - 1;
        wait(b_pvdone + 8 * (last & 1), (last >> 1) & 1, 4);
      }
      if (kGroups == 2) nan_notes[group * 128 + token] = nan_rows;
      if (vote_all(!ok)) break;
      tc_fence_after();
      // a group that had no page of the unit (it was cut to one) has sums of zero, references unset and no O^T
      bool has[kGroups];
      int2 copy[kGroups];
#pragma unroll
      for (int x = 0; x < kGroups; ++x) copy[x] = kGroups == 2 ? side_notes[x] : make_int2((turn - 1) & 1, side);
#pragma unroll
      for (int x = 0; x < kGroups; ++x) has[x] = kGroups == 1 || t1 - t0 >= 2 || ((it - 1) & 1) == x;
      if (kGroups == 2) nan_rows |= nan_notes[(group ^ 1) * 128 + token];
      const bool whole_unit = t0 == 0 && t1 == v.tiles;
      const int64_t slot = 2 * static_cast<int64_t>(blockIdx.x) + (t0 > 0 ? 0 : 1);
#pragma unroll
      for (int g = 0; g < N; g += 8) {
        if (g >= rows) break;
        if (kGroups == 2 && ((g >> 3) & 1) != group) continue;  // the groups share the rows
        float o[8], sum[8], base[8];
#pragma unroll
        for (int x = 0; x < kGroups; ++x) {
          uint32_t part[kPTerms][8];
#pragma unroll
          for (int y = 0; y < kPTerms; ++y) tmem_ld_32x8(t_all + x * kOCols + y * N + g, part[y]);
          float lx[8], rx[8];
          const float* sx = maxima + x * 8 * N + copy[x].x * 4 * N + g;
          load8(sx, lx);
#pragma unroll
          for (int q = 1; q < 4; ++q) {
            float w[8];
            load8(sx + q * N, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) lx[j] += w[j];
          }
          load8(refs + x * 2 * N + copy[x].y * N + g, rx);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            float ox = __uint_as_float(part[kPTerms - 1][j]);
#pragma unroll
            for (int y = kPTerms - 2; y >= 0; --y) ox = fmaf(ox, 1.f / kPStep, __uint_as_float(part[y][j]));
            if (!has[x]) {
              ox = 0.f;
              lx[j] = 0.f;
              rx[j] = kUnset;
            }
            if (x == 0) {
              o[j] = ox;
              sum[j] = lx[j];
              base[j] = rx[j];
            } else {
              const float m = fmaxf(base[j], rx[j]), f0 = exp2_approx(base[j] - m), f1 = exp2_approx(rx[j] - m);
              o[j] = fmaf(o[j], f0, ox * f1);
              sum[j] = fmaf(sum[j], f0, lx[j] * f1);
              base[j] = m;
            }
          }
        }
        if (nan_rows != 0) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if ((nan_rows >> (g + j)) & 1u) o[j] = __uint_as_float(0x7fc00000u);
        }
        if (whole_unit) {
          T res[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) res[j] = static_cast<T>(sum[j] == 0.f ? 0.f : __fdividef(o[j], sum[j]));
          int i = g / p.group, in_group = g - i * p.group;
          T* out = static_cast<T*>(p.o) + (v.lo + i) * p.o_tok + (static_cast<int64_t>(cur.h) * p.group + in_group) * p.o_head + token;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if (g + j < rows && token < DIM) *out = res[j];
            out += p.o_head;
            if (++in_group == p.group) {
              in_group = 0;
              out += p.o_tok - p.group * p.o_head;
            }
          }
        } else {
          if (token < DIM) {
#pragma unroll
            for (int j = 0; j < 8; ++j) p.part_o[(slot * N + g + j) * DIM + token] = o[j];
          }
          if (token == 0) {
#pragma unroll
            for (int j = 0; j < 8; ++j) p.part_ml[slot * N + g + j] = make_float2(base[j], sum[j]);
          }
        }
      }
      tc_fence_before();
      if (t0 == 0 && t1 < v.tiles) {
        // the unit begins here and goes on behind this block
        const int64_t unit_end = number_at + numbers(v);
        rec = make_int4(v.lo, cur.h, v.n, static_cast<int>((unit_end * blocks - 1) / total));
      }
      number_at += numbers(v);
      if (left > 0 && !next_unit(p, cur)) break;
    }
    if (!ok && lane == 0) *p.status = kRoleEpilogue * 1000 + site;
    if (work && at == 0) p.record[blockIdx.x] = abort_flag[0] ? make_int4(-1, 0, 0, 0) : rec;
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, Sh::kTmem);
  }
}

// Adds the parts of a unit that was cut by a block's range, in block order.  Block (i, y): rows 4 y .. 4 y + 3 of the unit that
// block i of the kernel above left unfinished.
template <typename T, int DIM>
__global__ void __launch_bounds__(4 * DIM) tg_attention_join_kernel(const AttentionParams p, int rows_padded) {
  griddep_wait();
  griddep_launch_dependents();
  const int4 rec = p.record[blockIdx.x];
  const int r = blockIdx.y * 4 + threadIdx.x / DIM, d = threadIdx.x % DIM;
  if (rec.x < 0 || r >= rec.z * p.group) return;
  const int first = blockIdx.x, last = min(rec.w, static_cast<int>(gridDim.x) - 1);
  const int64_t head = (2 * static_cast<int64_t>(first) + 1) * rows_padded + r;  // the first part: slot 1 of its block
  // eight parts at a time, their loads in flight together
  float m = -1e30f, l = 0.f, o = 0.f;
  for (int i0 = first; i0 <= last; i0 += 8) {
    float2 ml[8];
    float x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int i = min(i0 + k, last);
      const int64_t at = i == first ? head : 2 * static_cast<int64_t>(i) * rows_padded + r;
      ml[k] = p.part_ml[at];
      x[k] = p.part_o[at * DIM + d];
      if (i0 + k > last) {
        ml[k] = make_float2(-1e30f, 0.f);
        x[k] = 0.f;
      }
    }
    float top = m;
#pragma unroll
    for (int k = 0; k < 8; ++k) top = fmaxf(top, ml[k].x);
    const float shrink = exp2f(m - top);
    l *= shrink;
    o *= shrink;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float f = exp2f(ml[k].x - top);
      l = fmaf(ml[k].y, f, l);
      o = fmaf(x[k], f, o);
    }
    m = top;
  }
  const int i = r / p.group;
  static_cast<T*>(p.o)[(rec.x + i) * p.o_tok + (rec.y * p.group + r - i * p.group) * p.o_head + d] = static_cast<T>(l == 0.f ? 0.f : o / l);
}

template <typename T, int DIM, int N>
cudaError_t launch_n(const CUtensorMap& tmK, const CUtensorMap& tmV, const AttentionParams& p, int blocks, cudaStream_t stream) {
  constexpr int kTerms = kTermsOf<T>;
  using Sh = Shape<DIM, N, kTerms>;
  auto kernel = tg_attention_few_rows_kernel<T, DIM, N>;
  static bool set[64] = {};  // per device; set again at worst
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (!set[dev & 63]) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::kSmem);
    if (e != cudaSuccess) return e;
    set[dev & 63] = true;
  }
  e = launch_pdl(kernel, dim3(blocks), dim3(Sh::kThreads), Sh::kSmem, stream, tmK, tmV, p);
  if (e != cudaSuccess) return e;
  return launch_pdl(tg_attention_join_kernel<T, DIM>, dim3(blocks, (p.max_q_len * p.group + 3) / 4), dim3(4 * DIM), 0, stream, p, N);
}

template <typename T, int DIM>
cudaError_t launch_rows(const CUtensorMap& tmK, const CUtensorMap& tmV, const AttentionParams& p, int n, int blocks, cudaStream_t stream) {
  return n == 16 ? launch_n<T, DIM, 16>(tmK, tmV, p, blocks, stream) : launch_n<T, DIM, 32>(tmK, tmV, p, blocks, stream);
}

}  // namespace

int few_rows_padded(int rows) { return rows <= 16 ? 16 : 32; }

int few_rows_blocks(int dim, int rows_padded, bool bf16, int num_sms) {
  static_assert(Shape<128, 16, 2>::kBlocksPerSm == 2 && Shape<64, 16, 3>::kBlocksPerSm == 2 && Shape<128, 16, 3>::kBlocksPerSm == 1 &&
                Shape<64, 32, 2>::kBlocksPerSm == 1, "the rule below");
  return num_sms * (rows_padded == 16 && (bf16 || dim == 64) ? 2 : 1);
}

uint64_t few_rows_workspace(int dim, int rows_padded, int blocks) {
  const uint64_t parts = 2ull * blocks * rows_padded;
  return parts * dim * 4 + parts * 8 + 16ull * blocks;
}

cudaError_t launch_attention_few_rows(const CUtensorMap& tmK, const CUtensorMap& tmV, const AttentionParams& p, int rows_padded,
                                      int blocks, bool bf16, cudaStream_t stream) {
  if (bf16)
    return p.c.dim == 128 ? launch_rows<__nv_bfloat16, 128>(tmK, tmV, p, rows_padded, blocks, stream)
                          : launch_rows<__nv_bfloat16, 64>(tmK, tmV, p, rows_padded, blocks, stream);
  return p.c.dim == 128 ? launch_rows<__half, 128>(tmK, tmV, p, rows_padded, blocks, stream)
                        : launch_rows<__half, 64>(tmK, tmV, p, rows_padded, blocks, stream);
}

}  // namespace tg
