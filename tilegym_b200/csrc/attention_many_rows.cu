// Attention over the paged e4m3 cache for many rows: prompts, whole or in chunks.
//
// A block owns two tiles of 128 rows of one (sequence, cache head); a row is a (token, query head of the group) pair, so a
// key or value page that is loaded once serves the whole group.
//
//   S [128 rows, 128 tokens] = Q . K^T      kind::f8f6f4 on the cached bytes, q split into e4m3 terms (bf16: two hold it
//                                           exactly) that the accumulator sums: the time of one 16-bit product, no conversion of K
//   p = 2^(S * scale * log2 e + log2 v_scale - ref)   thread = row: no exchange between threads at all
//   O [128 rows, dim]       += P . V        kind::f16: P in f16 from TMEM, V converted e4m3 -> f16 (exact) by four warps once
//                                           per page for both tiles
//
// The work goes by half pages (64 tokens): TMEM holds O of both tiles (2 x 128 columns) and two S buffers of 64 columns for
// each, P taking the place of the S it came from, so that the next scores are there when a softmax is done with the last
// and the tensor core never waits for one tile alone.  `ref` is a running maximum, less 8, that
// moves only when a p would exceed 2^15 (f16 has room for that), which is when O is rescaled in TMEM.
// Few blocks (a chunk of a prompt on a long cache, few heads) leave most SMs idle: there `splits` blocks share a block's pages,
// each at least kMinPages, and a joining kernel adds their parts in order.
// Warp 0 copies pages, warps 1 and 2 issue the tiles' score products and warp 3 the value products (a warp that issues is
// held up until the tensor core has nearly caught up and then needs a few hundred clocks to find its next barriers ready:
// with one warp for all the tensor core was idle 60 % of the time, with two 45 %), warps 4-7 convert values, warps 8-11 and 12-15 are the tiles' softmax.
//
// Bound: the chain scores -> softmax -> product of a half page (about 1700 clocks for both tiles; the products need 1250, the
// exponentials 1024).  Measured (bf16, 32 heads on 8 of 128): 4 prompts of 300-2500 tokens on up to 5000 cached 250 us
// (765 TFLOP/s of 1631 measured for a 16-bit GEMM; 351 with whole pages and one issuing warp), one of 4096 174 us.
#include <cstdio>

#include "tg_attention.cuh"

namespace tg {
namespace {

constexpr int kThreads = 512;
constexpr int kRegsLaunch = 128, kRegsOther = 72, kRegsSoftmax = 184;
constexpr int kHalf = kPage / 2;  // tokens of a step
constexpr int kPoly = 5;
constexpr int kMinPages = 4;  // of a part: joining takes as long as three or four pages
constexpr float kUnset = -1e30f;  // the reference of a row that has not seen a token yet
// A row's largest p is 2^8 when ref is set and may reach 2^15 before ref moves (f16 ends at 2^16): f16 keeps its relative
// rounding down to 2^-22 of the largest.  A first token with most of the weight leaves the rest of a long cache there.
constexpr float kNominal = 8.f, kLimit = 15.f;

template <int DIM, int TERMS>
struct Shape {
  static constexpr int kTile = DIM * kPage;      // bytes of a key or value page
  static constexpr int kQ = TERMS * 128 * DIM;   // a tile's query terms
  static constexpr int kV16 = 2 * kTile;
  static constexpr int kStages = (227 * 1024 - 1024 - 2048 - 2 * kQ - 2 * kV16) / (2 * kTile) > 4
                                     ? 4 : (227 * 1024 - 1024 - 2048 - 2 * kQ - 2 * kV16) / (2 * kTile);
  static constexpr int kSmem = 1024 + kStages * 2 * kTile + 2 * kV16 + 2 * kQ + 2048;
  static_assert(kStages >= 2, "two pages in flight");
};

// D[tmem] (+)= A[tmem, f16] . B[smem, f16]^T, K = 16
__device__ __forceinline__ void mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
      "}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_st_32x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};"
      ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
      "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
      "r"(r[31]), "r"(taddr)
      : "memory");
}

__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile uint32_t* abort_flag) {
  return __all_sync(0xffffffffu, mbar_wait<false>(bar, parity, abort_flag));
}

__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }  // 0x80 at every 0x7f

__device__ __forceinline__ void to_f16(uint32_t w, uint32_t& a, uint32_t& b) {
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(a) : "h"(static_cast<uint16_t>(w)));
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(b) : "h"(static_cast<uint16_t>(w >> 16)));
}

// maxima that a NaN gets through: the polynomial below would swallow one
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// 2^x of a pair without the special-function unit: x = n + f with |f| <= 1/2, 2^f by a polynomial of degree 4 (fitted to the
// relative error over that range, 2.6e-6 at most), n added to the exponent.  x <= 100; below -126 the result is 2^-126 or so,
// which f16 rounds to zero (its share of the 32-bit sum is as small).  A NaN is taken for -126: the row's maximum has seen to it.
__device__ __forceinline__ float2 exp2_pair(float2 x) {
  const float2 magic = make_float2(12582912.f, 12582912.f), minus = make_float2(-12582912.f, -12582912.f);
  x.x = fmaxf(x.x, -126.f);
  x.y = fmaxf(x.y, -126.f);
  const float2 t = __fadd2_rn(x, magic);  // n in the low bits
  const float2 n = __fadd2_rn(t, minus);
  const float2 f = __fadd2_rn(x, make_float2(-n.x, -n.y));
  float2 r = __ffma2_rn(make_float2(0.0095701f, 0.0095701f), f, make_float2(0.05591787f, 0.05591787f));
  r = __ffma2_rn(r, f, make_float2(0.24024745f, 0.24024745f));
  r = __ffma2_rn(r, f, make_float2(0.69312181f, 0.69312181f));
  r = __ffma2_rn(r, f, make_float2(0.99999926f, 0.99999926f));
  r.x = __uint_as_float(__float_as_uint(r.x) + (__float_as_uint(t.x) << 23));
  r.y = __uint_as_float(__float_as_uint(r.y) + (__float_as_uint(t.y) << 23));
  return r;
}

// Parts that the pages of 256 rows are divided into.
__device__ __forceinline__ int parts_of(const AttentionParams& p, const SeqView& v) { return max(min(p.splits, v.tiles / kMinPages), 1); }

template <typename T, int DIM, bool kSplit>
__global__ void __launch_bounds__(kThreads, 1)
    tg_attention_many_rows_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                                  const __grid_constant__ AttentionParams p, int token_tiles, int tile_tokens) {
  constexpr int kTerms = std::is_same<T, __half>::value ? 3 : 2;
  using Sh = Shape<DIM, kTerms>;
  constexpr int kStages = Sh::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* v16_smem = smem + kStages * 2 * Sh::kTile;
  uint8_t* q_smem = v16_smem + 2 * Sh::kV16;
  uint8_t* misc = q_smem + 2 * Sh::kQ;
  uint64_t* bars = reinterpret_cast<uint64_t*>(misc);
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(misc + 512);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(misc + 528);
  uint32_t* nan_flag = reinterpret_cast<uint32_t*>(misc + 532);
  float* rowmul = reinterpret_cast<float*>(misc + 1024);  // [2][128]
  const uint32_t bar0 = smem_u32(bars);
  const uint32_t b_kfull = bar0, b_kempty = b_kfull + 8 * kStages, b_vfull = b_kempty + 8 * kStages, b_vempty = b_vfull + 8 * kStages,
                 b_hfull = b_vempty + 8 * kStages, b_hempty = b_hfull + 16, b_qready = b_hempty + 16;
  // by tile and buffer: + 16 * tile + 8 * buffer
  const uint32_t b_sfull = b_qready + 16, b_pready = b_sfull + 32, b_pvdone = b_pready + 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (warp == 0) {
    if (elect_one()) {
      prefetch_tmap(&tmK);
      prefetch_tmap(&tmV);
    }
    if (lane == 0) {
      for (int i = 0; i < kStages; ++i) {
        mbar_init(b_kfull + 8 * i, 1);
        mbar_init(b_kempty + 8 * i, 2);
        mbar_init(b_vfull + 8 * i, 1);
        mbar_init(b_vempty + 8 * i, 4);
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(b_hfull + 8 * i, 4);
        mbar_init(b_hempty + 8 * i, 1);
        mbar_init(b_qready + 8 * i, 4);
      }
      for (int i = 0; i < 4; ++i) {
        mbar_init(b_sfull + 8 * i, 1);
        mbar_init(b_pready + 8 * i, 4);
        mbar_init(b_pvdone + 8 * i, 1);
      }
      init_abort_flag(abort_flag, p.wait_limit_us);
      *nan_flag = 0;
      fence_mbar_init();
    }
  } else if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  griddep_wait();
  griddep_launch_dependents();
  // later tokens see more: their blocks come first
  const int whole_block = kSplit ? blockIdx.x / p.splits : blockIdx.x, split = kSplit ? blockIdx.x - whole_block * p.splits : 0;
  const int head = whole_block % p.c.heads;
  const int tile = token_tiles - 1 - whole_block / p.c.heads;
  int first;
  const int b = find_sequence(p.c.cu, p.c.seqs, tile, 2 * tile_tokens, 1, first);
  SeqView v = {};
  if (tile >= first) v = view_sequence(p, b, (tile - first) * 2 * tile_tokens, 2 * tile_tokens);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // this block's part of the pages, from number t0 on
  const int parts = kSplit ? parts_of(p, v) : 1;
  const int t0 = kSplit && split < parts ? static_cast<int>(static_cast<int64_t>(v.tiles) * split / parts) : 0;
  const int pages = v.n <= 0 || split >= parts ? 0 : kSplit ? static_cast<int>(static_cast<int64_t>(v.tiles) * (split + 1) / parts) - t0 : v.tiles;
  const int tiles = v.n > tile_tokens ? 2 : 1;  // that have rows
  bool ok = true;
  int site = 0;

  // Registers: the warps that copy, multiply and convert give up what the softmax warps, which hold half a row of S, take.
  static_assert(2 * kRegsOther + 2 * kRegsSoftmax <= 4 * kRegsLaunch && kRegsLaunch * kThreads <= 65536, "within what the block was launched with");
  if (warp < 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
    if (pages == 0 || (warp == 2 && tiles == 1)) {
      // no rows: a number of the ragged numbering that nobody has; or none in the second tile
    } else if (warp == 0) {
    // ------------------------------------------------------------------------------------------ copies
    const int rows_k = p.c.pages * p.c.heads * kPage, rows_v = p.c.pages * p.c.heads * DIM;
    int issued = 0;
    for (int base = 0; base < pages && ok; base += 32) {
      const int page = base + lane < pages ? v.page_of(t0 + base + lane) : p.c.max_pages;
      int phys = page < p.c.max_pages ? p.c.table[b * p.c.table_pitch + page] : -1;
      if (phys < 0 || phys >= p.c.pages) phys = -1;
      for (int i = 0; i < min(32, pages - base); ++i, ++issued) {
        const int stage = issued % kStages;
        const uint32_t parity = ((issued / kStages) & 1) ^ 1;
        const int ph = __shfl_sync(0xffffffffu, phys, i);
        // a page that is not there: a box behind the end of the cache, which reads as zeros
        const int yk = ph >= 0 ? (ph * p.c.heads + head) * kPage : rows_k, yv = ph >= 0 ? (ph * p.c.heads + head) * DIM : rows_v;
        const uint32_t dst = smem_u32(smem + stage * 2 * Sh::kTile);
        if (!warp_wait(b_kempty + 8 * stage, parity, abort_flag)) {
          ok = false;
          site = 1;
          break;
        }
        if (elect_one()) {
          mbar_arrive_expect_tx(b_kfull + 8 * stage, Sh::kTile);
          tma_load_2d(dst, &tmK, b_kfull + 8 * stage, 0, yk);
        }
        __syncwarp();
        if (!warp_wait(b_vempty + 8 * stage, parity, abort_flag)) {
          ok = false;
          site = 2;
          break;
        }
        if (elect_one()) {
          mbar_arrive_expect_tx(b_vfull + 8 * stage, Sh::kTile);
          tma_load_2d(dst + Sh::kTile, &tmV, b_vfull + 8 * stage, 0, yv);
        }
        __syncwarp();
      }
    }
    if (!ok) {
      if (lane == 0) *p.status = kRoleProducer * 1000 + site;
      // copies still in flight land before the block leaves (a bounded number of parked tries each; the page at which it
      // stopped may have its keys under way)
      for (int i = max(issued - kStages, 0); i <= issued; ++i) {
        const uint32_t parity = (i / kStages) & 1;
        if (i < issued || site == 2)
          for (int tries = 0; tries < 1000 && !mbar_try_wait(b_kfull + 8 * (i % kStages), parity); ++tries) {
          }
        if (i < issued)
          for (int tries = 0; tries < 1000 && !mbar_try_wait(b_vfull + 8 * (i % kStages), parity); ++tries) {
          }
      }
    }
    } else if (warp < 4) {
    // ------------------------------------------------------------------------------------------ products
    constexpr uint32_t idesc_s = make_idesc_e4m3_f32(128, kHalf);
    constexpr uint32_t idesc_o = make_idesc_e4m3_f32(128, DIM);  // the same fields: format 0 is f16 in kind::f16
    // every number that an address is made of comes from lane 0, so that it can live in uniform registers
    const uint32_t base = __shfl_sync(0xffffffffu, smem_u32(smem), 0), tm = __shfl_sync(0xffffffffu, tmem, 0);
    const uint32_t v_addr = base + kStages * 2 * Sh::kTile, q_addr = v_addr + 2 * Sh::kV16;
    const int halves = 2 * __shfl_sync(0xffffffffu, pages, 0), active = __shfl_sync(0xffffffffu, tiles, 0);
    auto need = [&](uint32_t bar, uint32_t parity, int where) {
      if (ok && !warp_wait(bar, parity, abort_flag)) {
        ok = false;
        site = where;
      }
    };
    if (warp < 3) {
      // scores of half page h of this warp's tile, into buffer h & 1: behind the product that read P from there
      const int w = __shfl_sync(0xffffffffu, warp, 0) - 1;
      int stage = 0;
      uint32_t round = 0;
      need(b_qready + 8 * w, 0, 1);
#pragma unroll 1
      for (int h = 0; h < halves && ok; ++h) {
        const int buf = h & 1;
        if (buf == 0) need(b_kfull + 8 * stage, round, 2);
        if (h >= 2) need(b_pvdone + 16 * w + 8 * buf, ((h >> 1) & 1) ^ 1, 3);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t bd = rows_desc<DIM>(base + stage * 2 * Sh::kTile + buf * kHalf * DIM);
#pragma unroll
          for (int term = 0; term < kTerms; ++term) {
            const uint64_t ad = rows_desc<DIM>(q_addr + w * Sh::kQ + term * 128 * DIM);
#pragma unroll
            for (int k = 0; k < DIM / 32; ++k) mma_f8f6f4(tm + w * 128 + buf * kHalf, ad + 2 * k, bd + 2 * k, idesc_s, term + k > 0);
          }
          tc_commit(b_sfull + 16 * w + 8 * buf);
          if (buf == 1) {
            // the stage is free when both tiles have read it
            tc_commit(b_kempty + 8 * stage);
            if (active == 1) tc_commit(b_kempty + 8 * stage);
          }
        }
        __syncwarp();
        if (buf == 1 && ++stage == kStages) {
          stage = 0;
          round ^= 1u;
        }
      }
    } else {
#pragma unroll 1
      for (int h = 0; h < halves && ok; ++h) {
        const int j = h >> 1, buf = h & 1;
        if (buf == 0) need(b_hfull + 8 * (j & 1), (j >> 1) & 1, 4);
#pragma unroll 1
        for (int w = 0; w < active; ++w) {
          need(b_pready + 16 * w + 8 * buf, j & 1, 5);
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
            const uint64_t bd = make_kmajor_sw128_desc(v_addr + (j & 1) * Sh::kV16 + buf * Sh::kTile);
#pragma unroll
            for (int k = 0; k < kHalf / 16; ++k) mma_f16_ts(tm + 256 + w * 128, tm + w * 128 + buf * kHalf + k * 8, bd + 2 * k, idesc_o, h + k > 0);
            tc_commit(b_pvdone + 16 * w + 8 * buf);
            if (w == active - 1 && buf == 1) tc_commit(b_hempty + 8 * (j & 1));
          }
          __syncwarp();
        }
      }
    }
    if (!ok && lane == 0) *p.status = kRoleMma * 1000 + site;
    } else {
    // ------------------------------------------------------------------------------------------ values to f16
    const int t = (warp - 4) * 32 + lane;
    bool nan = false;
    // the queries pass through this space first
    for (int w = 0; w < tiles && ok; ++w) ok = warp_wait(b_qready + 8 * w, 0, abort_flag);
    for (int j = 0; j < pages && ok; ++j) {
      const int stage = j % kStages;
      if (!warp_wait(b_vfull + 8 * stage, (j / kStages) & 1, abort_flag) || !warp_wait(b_hempty + 8 * (j & 1), ((j >> 1) & 1) ^ 1, abort_flag)) {
        ok = false;
        break;
      }
      const uint8_t* src = smem + stage * 2 * Sh::kTile + Sh::kTile;
      uint8_t* dst = v16_smem + (j & 1) * Sh::kV16;
#pragma unroll 4
      for (int u = t; u < DIM * 8; u += 128) {
        const int d = u % DIM, c = u / DIM;  // sixteen tokens of one element: 16 bytes in, 32 out
        const uint4 w = *reinterpret_cast<const uint4*>(src + d * kPage + ((c ^ (d & 7)) << 4));
        uint32_t ww[4] = {w.x, w.y, w.z, w.w};
        if ((nan_bytes(w.x) | nan_bytes(w.y) | nan_bytes(w.z) | nan_bytes(w.w)) != 0) {
          // a NaN becomes zero here, and is of interest only where some row sees the token
          const int at = v.page_of(t0 + j) * kPage + c * 16;
#pragma unroll
          for (int x = 0; x < 16; ++x)
            if (((ww[x >> 2] >> (8 * (x & 3))) & 127u) == 127u && at + x < min(v.len, v.pos0 + v.n) &&
                (p.window == 0 || at + x > static_cast<int64_t>(v.pos0) - p.window || at + x < p.sinks))
              nan = true;
#pragma unroll
          for (int x = 0; x < 4; ++x) ww[x] &= ~((nan_bytes(ww[x]) >> 7) * 255u);
        }
        uint4 lo, hi;
        to_f16(ww[0], lo.x, lo.y);
        to_f16(ww[1], lo.z, lo.w);
        to_f16(ww[2], hi.x, hi.y);
        to_f16(ww[3], hi.z, hi.w);
        uint8_t* at = dst + (c >> 2) * Sh::kTile + d * 128;
        const int c2 = (c & 3) * 2;
        *reinterpret_cast<uint4*>(at + ((c2 ^ (d & 7)) << 4)) = lo;
        *reinterpret_cast<uint4*>(at + (((c2 + 1) ^ (d & 7)) << 4)) = hi;
      }
      if (nan) *reinterpret_cast<volatile uint32_t*>(nan_flag) = 1u;
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(b_hfull + 8 * (j & 1));
        mbar_arrive(b_vempty + 8 * stage);
      }
    }
    if (!ok && lane == 0) *p.status = kRoleProducer * 1000 + 3;
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    if (pages > 0 && (warp - 8) / 4 < tiles) {
    // ------------------------------------------------------------------------------------------ softmax: thread = row
    const int w = (warp - 8) / 4, quarter = warp & 3, row = quarter * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t t_s0 = tmem + w * 128 + lane_off, t_o = tmem + 256 + w * 128 + lane_off;
    const int i = w * tile_tokens + row / p.group, g = row % p.group;  // token of the block, head of the group
    const bool live = row < tile_tokens * p.group && i < v.n;
    const int pos = v.pos0 + i;
    // ---- queries: eight elements per thread, split into e4m3 terms under a power-of-two scale of their row (a short loop:
    // straight-line code that a block runs once is paid for in instruction fetches)
    {
      constexpr int kLanes = DIM / 8, kRows = 128 / kLanes;
      const int st = quarter * 32 + lane, e = (st % kLanes) * 8;
      // all copies first, into the space of the f16 values, which waits for the queries: one latency, no registers
      uint8_t* raw = v16_smem + w * Sh::kV16 + e * 2;
      const T* q0 = static_cast<const T*>(p.q) + static_cast<int64_t>(v.lo + w * tile_tokens) * p.q_tok + head * p.group * p.q_head + e;
      // (token, head of the group) of the row, stepped along with it
      int ti = (st / kLanes) / p.group, hg = st / kLanes - ti * p.group;
      const int step_t = kRows / p.group, step_h = kRows - step_t * p.group;
      const int tokens = min(tile_tokens, v.n - w * tile_tokens);
#pragma unroll 4
      for (int r = st / kLanes; r < 128; r += kRows) {
        if (ti < tokens)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(raw + r * (2 * DIM))), "l"(q0 + ti * p.q_tok + hg * p.q_head) : "memory");
        else
          *reinterpret_cast<uint4*>(raw + r * (2 * DIM)) = make_uint4(0, 0, 0, 0);
        ti += step_t;
        hg += step_h;
        if (hg >= p.group) {
          hg -= p.group;
          ++ti;
        }
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll 4
      for (int r = st / kLanes; r < 128; r += kRows) {
        const uint4 x = *reinterpret_cast<const uint4*>(raw + r * (2 * DIM));  // this thread's own copy
        const uint32_t ww[4] = {x.x, x.y, x.z, x.w};
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
          split_e4m3<kTerms>(f[2 * j] * inv, f[2 * j + 1] * inv, 1.f, term);
#pragma unroll
          for (int y = 0; y < kTerms; ++y) out[y][j >> 1] = (j & 1) ? out[y][j >> 1] | (term[y] << 16) : term[y];
        }
#pragma unroll
        for (int y = 0; y < kTerms; ++y)
          *reinterpret_cast<uint2*>(q_smem + w * Sh::kQ + y * 128 * DIM + swizzled<DIM>(r, e)) = make_uint2(out[y][0], out[y][1]);
        // a row that holds an infinity or NaN has no answer
        if (e == 0) rowmul[w * 128 + r] = top >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : sc * p.scale * 1.4426950408889634f;
      }
      fence_proxy_async_smem();
      asm volatile("barrier.cta.sync %0, 128;" ::"r"(1 + w) : "memory");  // the tile's four warps, none of which can fail here
      if (lane == 0) mbar_arrive(b_qready + 8 * w);
    }
    const float mul = rowmul[w * 128 + row];
    // what all rows of the tile see
    const int tile_first = v.pos0 + w * tile_tokens, tile_last = v.pos0 + min(v.n, (w + 1) * tile_tokens) - 1;
    const int all_hi = min(v.len, tile_first + 1);
    const int all_lo = p.window > 0 ? static_cast<int>(max(static_cast<int64_t>(tile_last) - p.window + 1, int64_t(0))) : 0;
    const int row_hi = min(v.len, pos + 1);
    const int row_lo = p.window > 0 ? static_cast<int>(max(static_cast<int64_t>(pos) - p.window + 1, int64_t(0))) : 0;
    // page numbers two pages ahead, scales one: nothing here waits for a load that it has just issued
    auto page_entry = [&](int j) {
      const int page = j < pages ? v.page_of(t0 + j) : p.c.max_pages;
      return page < p.c.max_pages ? p.c.table[b * p.c.table_pitch + page] : -1;
    };
    auto scales = [&](int phys, float& ks, float& vs) {
      ks = vs = 1.f;
      if (phys >= 0 && phys < p.c.pages) {
        ks = p.c.ks[static_cast<int64_t>(phys) * p.c.heads + head];
        vs = p.c.vs[static_cast<int64_t>(phys) * p.c.heads + head];
      }
    };
    float ref = kUnset, l = 0.f, ks, vs, ks1, vs1;
    int entry = page_entry(0), entry1 = page_entry(1);
    scales(entry, ks, vs);
    for (int j = 0; j < pages && ok; ++j) {
      scales(entry1, ks1, vs1);
      const int entry2 = page_entry(j + 2);
      const bool here = entry >= 0 && entry < p.c.pages;
      float f = mul * ks;
      // a factor that is no positive number (a row of q or a scale with an infinity or NaN) belongs to the tokens that the row
      // sees, but -inf * f of the hidden ones has to stay -inf
      if (f == 0.f) f = 1e-38f;
      const bool odd = !(f > 0.f && f < INFINITY);
      if (odd) f = 1.f;
      // log2 and reciprocal of the page's scale: a power of two where the cache was written by this library
      const uint32_t vb = __float_as_uint(vs);
      float lv, inv_vs;
      if ((vb & 0x807fffffu) == 0 && vb >= 0x00800000u && vb < 0x7e800000u) {
        lv = static_cast<float>(static_cast<int>(vb >> 23) - 127);
        inv_vs = pow2_reciprocal(vs);
      } else {
        lv = log2f(vs);
        inv_vs = 1.0f / vs;
      }
#pragma unroll 1
      for (int half = 0; half < 2; ++half) {
        const int base = v.page_of(t0 + j) * kPage + half * kHalf;
        const bool whole = here && base + kHalf <= all_hi && (base >= all_lo || base + kHalf <= p.sinks);
        const uint32_t t_s = t_s0 + half * kHalf;
        if (!warp_wait(b_sfull + 16 * w + 8 * half, j & 1, abort_flag)) {
          ok = false;
          site = 1;
          break;
        }
        tc_fence_after();
        uint32_t s[2][32];
        tmem_ld_32x32(t_s, s[0]);
        tmem_ld_32x32(t_s + 32, s[1]);
        tmem_ld_wait();
        if (!whole) {
          const int hi = here ? row_hi - base : 0, lo = row_lo - base, sink = p.sinks - base;
#pragma unroll
          for (int t = 0; t < kHalf; ++t)
            if (t >= hi || (t < lo && t >= sink)) s[t >> 5][t & 31] = 0xff800000u;
        }
        float mx[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          mx[c] = __uint_as_float(s[c >> 1][(c & 1) * 16]);
#pragma unroll
          for (int k = 1; k < 15; k += 2)
            mx[c] = max3(mx[c], __uint_as_float(s[c >> 1][(c & 1) * 16 + k]), __uint_as_float(s[c >> 1][(c & 1) * 16 + k + 1]));
        }
        auto last = [&](int c) { return __uint_as_float(s[c >> 1][(c & 1) * 16 + 15]); };
        mx[0] = max3(mx[0], last(0), last(1));
        mx[1] = max3(mx[1], last(2), last(3));
        mx[2] = max3(mx[2], mx[3], mx[0]);
        const float most = max3(mx[1], mx[2], mx[2]), top = fmaf(most, f, lv);
        // the row sees a NaN (the sum keeps it)
        if (most != -INFINITY && (odd || !(top < INFINITY))) l = __uint_as_float(0x7fc00000u);
        const bool move = top > ref + (ref == kUnset ? 0.f : kLimit);
        if (__any_sync(0xffffffffu, move)) {
          const float now = move ? top - kNominal : ref, shrink = exp2_approx(ref - now);
          ref = now;
          l *= shrink;
          if (j + half > 0) {
            // not before the product of the half page in front is done
            const int h = 2 * j + half - 1;
            if (!warp_wait(b_pvdone + 16 * w + 8 * (h & 1), (h >> 1) & 1, abort_flag)) {
              ok = false;
              site = 2;
              break;
            }
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < DIM; c += 32) {
              uint32_t o[32];
              tmem_ld_32x32(t_o + c, o);
              tmem_ld_wait();
#pragma unroll
              for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * shrink);
              tmem_st_32x32(t_o + c, o);
            }
            tmem_st_wait();
          }
        }
        const float shift = lv - ref;
        // every kPoly-th pair takes the polynomial: 16 exponentials a clock and SM are what bounds this loop
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        const float2 f2 = make_float2(f, f), shift2 = make_float2(shift, shift);
        uint32_t pk[32];
#pragma unroll
        for (int k = 0; k < 32; ++k) {
          const int c = k >> 4, e = (k & 15) * 2;
          const float2 z = __ffma2_rn(make_float2(__uint_as_float(s[c][e]), __uint_as_float(s[c][e + 1])), f2, shift2);
          const float2 pr = k % kPoly == kPoly - 1 ? exp2_pair(z) : make_float2(exp2_approx(z.x), exp2_approx(z.y));
          sum[k & 1] = __fadd2_rn(sum[k & 1], pr);
          pk[k] = pack_pair<__half>(pr.x, pr.y);
        }
        tmem_st_32x32(t_s, pk);
        // the sums take p as it is, in 32 bits
        l = fmaf((sum[0].x + sum[0].y) + (sum[1].x + sum[1].y), inv_vs, l);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(b_pready + 16 * w + 8 * half);
      }
      entry = entry1;
      ks = ks1;
      vs = vs1;
      entry1 = entry2;
    }
    if (ok && !warp_wait(b_pvdone + 16 * w + 8, (pages - 1) & 1, abort_flag)) {
      ok = false;
      site = 3;
    }
    if (ok) {
      tc_fence_after();
      // a NaN among the values was kept from the products: it belongs to the rows that see its token
      uint32_t bad[4] = {0, 0, 0, 0};
      if (*reinterpret_cast<volatile uint32_t*>(nan_flag) != 0) {
        for (int j = 0; j < pages; ++j) {
          const int ph = page_entry(j), base = v.page_of(t0 + j) * kPage;
          if (ph < 0 || ph >= p.c.pages) continue;
          const uint8_t* src = p.c.v + (static_cast<int64_t>(ph) * p.c.heads + head) * (kPage * DIM);
          for (int u = 0; u < DIM * 8; ++u) {
            const uint4 w = reinterpret_cast<const uint4*>(src)[u];
            const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
            const int d = u >> 3, t0 = base + (u & 7) * 16;
#pragma unroll
            for (int x = 0; x < 16; ++x)
              if (((ww[x >> 2] >> (8 * (x & 3))) & 127u) == 127u && t0 + x < row_hi && (t0 + x >= row_lo || t0 + x < p.sinks)) {
#pragma unroll
                for (int y = 0; y < 4; ++y)
                  if (y == (d >> 5)) bad[y] |= 1u << (d & 31);
              }
          }
        }
        __syncwarp();
      }
      // a row that has seen nothing: the polynomial's 2^-126 of hidden places is no sum (a NaN stays: the row has seen one)
      if (ref == kUnset && l == l) l = 0.f;
      const float inv = l == 0.f ? 0.f : 1.0f / l;
      const int64_t slot = static_cast<int64_t>(blockIdx.x) * 256 + w * 128 + row;
      if (kSplit && parts > 1) p.part_ml[slot] = make_float2(ref, l);
      T* out = static_cast<T*>(p.o) + static_cast<int64_t>(v.lo + i) * p.o_tok + (head * p.group + g) * p.o_head;
#pragma unroll 1
      for (int c = 0; c < DIM; c += 32) {
        uint32_t o[32];
        tmem_ld_32x32(t_o + c, o);
        tmem_ld_wait();
        const uint32_t nan = c < 64 ? (c < 32 ? bad[0] : bad[1]) : (c < 96 ? bad[2] : bad[3]);
        if (nan != 0) {
#pragma unroll
          for (int k = 0; k < 32; ++k)
            if ((nan >> k) & 1u) o[k] = 0x7fc00000u;
        }
        if (kSplit && parts > 1) {
          float4* part = reinterpret_cast<float4*>(p.part_o + slot * DIM + c);
#pragma unroll
          for (int k = 0; k < 32; k += 4)
            part[k / 4] = make_float4(__uint_as_float(o[k]), __uint_as_float(o[k + 1]), __uint_as_float(o[k + 2]), __uint_as_float(o[k + 3]));
        } else if (live) {
#pragma unroll
          for (int k = 0; k < 32; k += 8) {
            uint32_t r[4];
#pragma unroll
            for (int y = 0; y < 4; ++y)
              r[y] = l == 0.f ? 0u : pack_pair<T>(__uint_as_float(o[k + 2 * y]) * inv, __uint_as_float(o[k + 2 * y + 1]) * inv);
            *reinterpret_cast<uint4*>(out + c + k) = make_uint4(r[0], r[1], r[2], r[3]);
          }
        }
      }
      tc_fence_before();
    }
    if (!ok && lane == 0) *p.status = kRoleEpilogue * 1000 + site;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Adds the parts of a block in order: a warp per row, a lane DIM / 32 elements.
template <typename T, int DIM>
__global__ void __launch_bounds__(256) tg_attention_join_parts_kernel(const __grid_constant__ AttentionParams p, int token_tiles, int tile_tokens) {
  griddep_wait();
  griddep_launch_dependents();
  constexpr int E = DIM / 32;
  const int lane = threadIdx.x & 31, row = blockIdx.y * 8 + (threadIdx.x >> 5);  // of 256
  const int head = blockIdx.x % p.c.heads, tile = token_tiles - 1 - blockIdx.x / p.c.heads;
  int first;
  const int b = find_sequence(p.c.cu, p.c.seqs, tile, 2 * tile_tokens, 1, first);
  if (tile < first) return;
  const SeqView v = view_sequence(p, b, (tile - first) * 2 * tile_tokens, 2 * tile_tokens);
  const int parts = parts_of(p, v), r = row & 127;
  const int i = (row >> 7) * tile_tokens + r / p.group, g = r % p.group;
  if (parts == 1 || r >= tile_tokens * p.group || i >= v.n) return;
  const int64_t slot0 = static_cast<int64_t>(blockIdx.x) * p.splits * 256 + row;
  const float2 ml = lane < parts ? p.part_ml[slot0 + lane * 256] : make_float2(kUnset, 0.f);
  const float f = exp2f(ml.x - redux_max(ml.x));
  float l = ml.y * f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
  float sum[E] = {};
#pragma unroll 4
  for (int k = 0; k < parts; ++k) {
    const float fk = __shfl_sync(0xffffffffu, f, k);
    const float* part = p.part_o + (slot0 + k * 256) * DIM + lane * E;
    float x[E];
    if constexpr (E == 4) {
      const float4 y = *reinterpret_cast<const float4*>(part);
      x[0] = y.x; x[1] = y.y; x[2] = y.z; x[3] = y.w;
    } else {
      const float2 y = *reinterpret_cast<const float2*>(part);
      x[0] = y.x; x[1] = y.y;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) sum[e] = fmaf(x[e], fk, sum[e]);
  }
  T* out = static_cast<T*>(p.o) + static_cast<int64_t>(v.lo + i) * p.o_tok + (head * p.group + g) * p.o_head + lane * E;
  const float inv = 1.0f / l;
#pragma unroll
  for (int e = 0; e < E; e += 2) *reinterpret_cast<uint32_t*>(out + e) = l == 0.f ? 0u : pack_pair<T>(sum[e] * inv, sum[e + 1] * inv);
}

template <typename T, int DIM, bool kSplit>
cudaError_t launch_split(const CUtensorMap& tmK, const CUtensorMap& tmV, const AttentionParams& p, cudaStream_t stream) {
  constexpr int kTerms = std::is_same<T, __half>::value ? 3 : 2;
  using Sh = Shape<DIM, kTerms>;
  auto kernel = tg_attention_many_rows_kernel<T, DIM, kSplit>;
  static bool set[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (!set[dev & 63]) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::kSmem);
    if (e != cudaSuccess) return e;
    set[dev & 63] = true;
  }
  const int tile_tokens = 128 / p.group, token_tiles = static_cast<int>(many_rows_tiles(p.tokens, p.c.seqs, p.group));
  const int64_t blocks = static_cast<int64_t>(token_tiles) * p.c.heads;
  if (blocks * p.splits > 0x7fffffff) return cudaErrorInvalidValue;
  e = launch_pdl(kernel, dim3(static_cast<unsigned>(blocks * p.splits)), dim3(kThreads), Sh::kSmem, stream, tmK, tmV, p, token_tiles, tile_tokens);
  if (e != cudaSuccess || !kSplit) return e;
  return launch_pdl(tg_attention_join_parts_kernel<T, DIM>, dim3(static_cast<unsigned>(blocks), 256 / 8), dim3(256), 0, stream, p, token_tiles, tile_tokens);
}

template <typename T, int DIM>
cudaError_t launch(const CUtensorMap& tmK, const CUtensorMap& tmV, const AttentionParams& p, cudaStream_t stream) {
  return p.splits > 1 ? launch_split<T, DIM, true>(tmK, tmV, p, stream) : launch_split<T, DIM, false>(tmK, tmV, p, stream);
}

}  // namespace

int64_t many_rows_tiles(int64_t tokens, int64_t seqs, int group) { return tokens / (2 * (128 / group)) + seqs; }

// As many parts as there are SMs for.  100 tokens on 32000, 32 heads on 8: 87 us, undivided 542; 500 tokens on 4000, 8 heads
// on 2: 33 and 88; 1000 tokens on 4000, 32 heads on 8, are 136 blocks and stay whole (99 us).
int many_rows_splits(int64_t tokens, int64_t seqs, int64_t heads, int group, int64_t max_pages, int num_sms) {
  const int64_t blocks = many_rows_tiles(tokens, seqs, group) * heads;
  const int64_t most = max_pages / kMinPages < 32 ? max_pages / kMinPages : 32, fit = blocks > 0 ? num_sms / blocks : 1;
  return static_cast<int>(fit < 2 || most < 2 ? 1 : fit < most ? fit : most);
}

uint64_t many_rows_workspace(int dim, int64_t blocks, int splits) { return splits == 1 ? 0 : 256ull * blocks * splits * (dim * 4 + 8); }

cudaError_t launch_attention_many_rows(const CUtensorMap& tmK, const CUtensorMap& tmV, const AttentionParams& p, bool bf16,
                                       cudaStream_t stream) {
  if (bf16)
    return p.c.dim == 128 ? launch<__nv_bfloat16, 128>(tmK, tmV, p, stream) : launch<__nv_bfloat16, 64>(tmK, tmV, p, stream);
  return p.c.dim == 128 ? launch<__half, 128>(tmK, tmV, p, stream) : launch<__half, 64>(tmK, tmV, p, stream);
}

}  // namespace tg
