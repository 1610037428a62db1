// Attention of a ragged batch's newest tokens over a paged latent cache (absorbed MLA: every head reads the
// same rows).
//
// Token t of sequence b (cu[b] <= t < cu[b+1], n_b of them) sits at position p = lens[b] - n_b + (t - cu[b]) and
// attends the cache rows j <= p (row j: row j % P of page table[b, j / P]); with a window, those with
// j > p - window or j < first.  out = sum_j e^(s_j - m) row_j[:512] / (sum_j e^(s_j - m) + e^(sink - m)) with
// s_j = scale q.row_j; a token that sees no row gives 0.
//
// A sequence's (token, head) pairs are rows of q, n_b * H of them in a run; a tile is 32 NB of them.  The rows
// a tile visits are numbered through: entry e < nf is row e (the first rows, where the window starts
// behind them), entry e >= nf row lo + e - nf.  A work item is a run of `rps` entries of one tile; every
// workgroup finds its item from the lengths itself (no plan launch, no host read): with few tiles rps is the
// smallest that gives every compute unit at most one item, with many it only cuts entries that one workgroup
// would be long busy with.  Tiles of several items leave (m, l, O) states that paged_merge_kernel joins.
//
// A workgroup is 8 waves of up to 256 registers, two per SIMD, and walks its entries in tiles of 32 rows, two
// roles with one barrier a tile between:
//   * score waves 0 .. NB-1: S^T = K Q^T of 32 q rows (v_mfma_f32_32x32x16_bf16, rows as M; the 32 q rows' Q^T
//     stays in 144 registers), online softmax with a lazy maximum, P in bf16 and the rescale factor to LDS (the products
//     take rows and probabilities of one type, and the rows are bf16: against 64 bits a result is off by 1.7e-3 to 2.2e-3
//     of its 2-norm, 1.7e-3 of that its own rounding);
//   * value waves 3 .. 7: O^T += V^T P^T (v_mfma_f32_32x32x16_bf16) of 3 or 4 blocks of 32 value columns and all
//     the tile's q rows, so each V^T fragment (ds_read_b64_tr_b16) is read by one wave and serves NB products.
//     Wave 3 shares its SIMD with value wave 7 instead of a score wave and takes four blocks, the others three.
// At NB = 3 the matrix pipes of SIMDs 0 .. 2 have 1152 + 576 cycles a tile (D = 576), SIMD 3 has 1344, and the LDS about
// 850 (6.8 KB a row at 256 bytes a cycle).  A form with 64 q rows on 12 waves of 168 registers (16 rows' Q^T a score
// wave) read 8.4 KB a row for two thirds of the products and was 11.6 ms where this one is 7.9.
// NB = 2 (64 q rows) where that makes no more tiles (tile_blocks).
//
// What bounds it, measured: a 2048-token chunk at 32 K (64 heads, D 576) 7.6 to 8.1 ms = 1120 to 1200 TFLOP/s, the matrix
// pipes (a large library product reaches 1261 on the card); a decode step of 32 sequences of 2 K to 32 K rows 149 us =
// 5.3 TB/s, HBM; drafts of 64 sequences over fp8 rows 110 us, the conversion to bf16 beside the products; a 4096-token
// prompt in a 128-row window 200 us, five row tiles an item behind Q's arrival and before the output's leaving (Q and
// out alone are 113 us of HBM); one token over 4 K rows 11.4 us and 5.5 us for the join, latencies.
//
// Rows come HBM -> LDS by DMA into a ring of four tiles, copies issued by the value waves (fp8 rows: loaded,
// converted, written).  Row numbers go through an LDS ring of 8 tiles that score wave 0 fills six tiles
// ahead, so a row list of any length costs one table read per row.
//
// Rows masked for some of a tile's q rows may hold anything (rows not yet written, pages of id -1 read as
// row 0): their probability is 0, and where a score of the tile is not finite the value waves take its
// values with their infinities and NaN as 0.  So a row seen with a score of -inf counts for nothing, whatever else
// is in its tile; one seen with +inf or NaN makes its q row's sum NaN.
#include "attn_common.h"

namespace smla_attn {
namespace {

typedef int32_t i32x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) i32x4_t lds_i32x4_t;
typedef __attribute__((address_space(3))) u32x2_t lds_u32x2_t;
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));

constexpr int kIdTiles = 8;        // tiles of the row-number ring
constexpr int kMinRows = 64;       // fewest entries of an item (one token over 4 K rows, with the join: 64 17.7 us, 128 18.3, 256 20.7)
constexpr int kMinRowsMany = 256;  // the same with more tiles than compute units
constexpr int kMinPart = 4096, kMostParts = 4, kMostItems = 16, kPartRows = 256;  // parts of many tiles (plan_rps)
constexpr int kHeader = 256;       // workspace bytes before the states
constexpr int kWaves = 8, kFirstValue = 3, kValueWaves = 5;
constexpr int kUnits = 16;         // blocks of 32 value columns

struct PagedArgs {
  const uint16_t* q;
  const void* pages;
  const float* page_scales;
  const int32_t *table, *lens, *cu, *granted;  // granted null: every sequence
  const float* sink;
  uint16_t* out;
  uint8_t* ws;
  int64_t ld_table;
  int T, H, B, P, n_pages, cols, window, first, cus, slots, fill;
  float scale;
};

// LDS layouts without bank conflicts (64 banks: 256 bytes an access cycle).  16-byte chunk ch of row r's columns 0..511 lies
// at chunk ch ^ row_swizzle(r) of its 1024 bytes: the 16 rows of a K read's cycle fall on 16 chunks, and the four
// rows of a transposed V read's (64 bytes each) on four groups of four.  Chunk ch of q row r's 64 bytes of P lies at
// ch ^ ((r >> 2) & 3).  Measured: 4.7 cycles a 1 KB read against 8.0 with swizzles that repeat every 128 bytes.
__device__ inline constexpr int row_swizzle(int r) { return ((r & 3) << 2) | ((r >> 2) & 3); }
__device__ inline constexpr int p_at(int r, int ch) { return 64 * r + 16 * (ch ^ ((r >> 2) & 3)); }

template <int D, int NB_>
struct GeoP {
  static constexpr int NB = NB_;
  static constexpr int TILEQ = 32 * NB;  // q rows of a tile
  static constexpr int ROWB = D * 2;
  static constexpr bool TAIL = D > 512;
  static constexpr int MAIN_BYTES = kTileRows * 1024;  // columns 0..511 of 32 rows, in swizzled 16-byte chunks
  static constexpr int TAIL_BYTES = TAIL ? kTileRows * 128 : 0;
  static constexpr int TILE_BYTES = MAIN_BYTES + TAIL_BYTES;
  static constexpr int NBUF = 4;
  static constexpr int PBUF = TILEQ * 64;  // 32 probabilities a q row (p_at)
  static constexpr int P_OFF = NBUF * TILE_BYTES;
  static constexpr int AL_OFF = P_OFF + 2 * PBUF;  // rescale factors; after the loop (m, l)
  static constexpr int IDS_OFF = AL_OFF + 2 * TILEQ * 4;
  static constexpr int FLAG_OFF = IDS_OFF + kIdTiles * kTileRows * 4;  // a flag per P buffer and score wave
  static constexpr int LDS_BYTES = FLAG_OFF + 2 * 4 * 4;
  static constexpr int NDMA = kTileRows + (TAIL ? kTileRows / 8 : 0);
  static constexpr int STATE_O = kUnits * NB * 2048;                     // bytes of a state's O^T
  static constexpr int STATE_F = TILEQ * 2 + kValueWaves * NB * 64;       // floats: (m, l), then scales
  static_assert(LDS_BYTES <= 160 * 1024, "LDS budget");
  static_assert(NB <= kFirstValue && NBUF >= 3, "roles; a tile scored, one consumed, one on its way");
  static_assert(kIdTiles >= NBUF + 4, "row numbers are written before their copies are issued");
};

__device__ inline uint32_t pack2(float a, float b) { return pack_bf16x2(a, b); }

// the bf16 pair with an infinite or NaN half set to 0
__device__ inline uint32_t finite2(uint32_t w) {
  const uint32_t lo = (w & 0x7f80u) == 0x7f80u ? 0u : w & 0xffffu;
  const uint32_t hi = (w & 0x7f800000u) == 0x7f800000u ? 0u : w & 0xffff0000u;
  return lo | hi;
}

// ---------------------------------------------------------------------------------------------
// The plan.  One lane per sequence, 64 at a time; every workgroup computes the same.
struct Seq {
  int beg, n, len;  // first token, tokens, cache rows
  int tiles, span;  // tiles of q rows; entries that a tile may visit
};

template <int TILEQ>
__device__ inline Seq load_seq(const PagedArgs& a, int b) {
  Seq s{0, 0, 0, 0, 0};
  if (b < a.B) {
    const int c0 = a.cu[b], c1 = a.cu[b + 1], len = a.lens[b], has = a.granted ? a.granted[b] : 1;
    s.beg = min(max(c0, 0), a.T);
    s.n = has ? max(min(c1, a.T) - s.beg, 0) : 0;
    s.len = max(len, 0);
    s.tiles = (int)(((uint32_t)s.n * (uint32_t)a.H + TILEQ - 1) / TILEQ);
    const int64_t cap = (int64_t)a.cols * a.P;
    int64_t span = s.len < cap ? s.len : cap;
    if (a.window > 0) {
      const int64_t w = (int64_t)a.window + a.first + (TILEQ + a.H - 1) / a.H;  // + 1 token - 1
      span = span < w ? span : w;
    }
    s.span = (int)span;
  }
  return s;
}

__device__ inline int ceil_div(int a, int b) { return (int)(((uint32_t)a + (uint32_t)b - 1) / (uint32_t)b); }
__device__ inline int splits_of(const Seq& s, int rps) { return max(1, ceil_div(s.span, rps)); }
__device__ inline int wave_sum_i(int v) { return __builtin_amdgcn_readlane(wave_incl_scan(v), 63); }

// Most entries per item (a multiple of 32; a sequence's splits are equal parts of its entries).  s0: sequences 0..63, kept in registers by the caller.
template <int TILEQ>
__device__ inline int plan_rps(const PagedArgs& a, const Seq& s0, int lane) {
  float work = 0.f;
  int tiles = 0, most = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const Seq s = b0 == 0 ? s0 : load_seq<TILEQ>(a, b0 + lane);
    work += wave_sum_dpp((float)s.tiles * (float)s.span);
    tiles += wave_sum_i(s.tiles);
    most = max(most, (int)wave_max_dpp((float)(s.tiles > 0 ? s.span / kTileRows + 1 : 0)));
  }
  if (tiles > a.cus) {
    // more tiles than compute units: items of at most half a unit's share
    const float share = work / (float)(2 * a.cus * kTileRows);
    const int best = max(kMinRowsMany / kTileRows, (int)fminf(share, 16777216.f) + 1);
    // (past 2 kMinPart entries, where plan_slots has slots for the parts; `most` is one more than whole tiles)
    if (most <= kMinPart / kTileRows * 2 || 2 * (int64_t)tiles > kMostItems * a.cus) return best * kTileRows;
    // few rounds of long tiles: parts of them fill the last round better; a part costs about kPartRows entries more
    float least = 0.f;
    int rps = best;
    for (int k = 1; k <= kMostParts && most / k >= kMinPart / kTileRows && k * tiles <= kMostItems * a.cus; k++) {
      const int unit = min(best, (most + k - 1) / k);
      int items = 0;
      for (int b0 = 0; b0 < a.B; b0 += 64) {
        const Seq s = b0 == 0 ? s0 : load_seq<TILEQ>(a, b0 + lane);
        items += wave_sum_i(s.tiles * splits_of(s, unit * kTileRows));
      }
      const float cost = (float)ceil_div(items, a.cus) * (work / (float)items + (float)kPartRows);
      if (k == 1 || cost < least) {
        least = cost;
        rps = unit;
      }
    }
    return rps * kTileRows;
  }
  // units of 32 entries: the fewest that give at most one item per compute unit
  int lo = max(kMinRows / kTileRows, (int)fminf(work / (float)(a.cus * kTileRows), 16777216.f));
  int hi = max(lo, most + (most >> 20) + 1);  // (most went through fp32)
  // (sum of tiles x ceil(span / rps) <= work / rps + tiles: enough where that fits; fp32 sums of at most 256 terms and their
  // quotient are off by under 1e-4 of it)
  if (tiles < a.cus) {
    const float fits = work / (float)((a.cus - tiles) * kTileRows) * 1.0001f;
    if (fits < (float)hi) hi = max(lo, (int)fits + 2);
  }
  while (lo < hi) {
    const int mid = lo + (hi - lo) / 2;
    int items = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
      const Seq s = b0 == 0 ? s0 : load_seq<TILEQ>(a, b0 + lane);
      items += wave_sum_i(s.tiles * splits_of(s, mid * kTileRows));
    }
    if (items <= a.cus) hi = mid;
    else lo = mid + 1;
  }
  return lo * kTileRows;
}

// Item w: its sequence, tile and split, and the state slot of the tile's first split.  false: no such item.
// by_tile: w counts tiles of split sequences instead (the merge's work).
struct Item {
  Seq s;
  int b, tile, split, nsplit, slot;
};
template <int TILEQ>
__device__ inline bool find_item(const PagedArgs& a, const Seq& s0, int lane, int rps, int w, bool by_tile, Item& it) {
  int before = 0, slots = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const Seq s = b0 == 0 ? s0 : load_seq<TILEQ>(a, b0 + lane);
    const int ns = splits_of(s, rps);
    const int states = ns > 1 ? s.tiles * ns : 0;
    const int mine = by_tile ? (ns > 1 ? s.tiles : 0) : s.tiles * ns;
    const int incl = wave_incl_scan(mine), sincl = wave_incl_scan(states);
    const uint64_t has = __builtin_amdgcn_ballot_w64(before + incl > w);
    if (has) {
      const int k = (int)__builtin_ctzll(has);
      it.b = b0 + k;
      it.s.beg = __builtin_amdgcn_readlane(s.beg, k);
      it.s.n = __builtin_amdgcn_readlane(s.n, k);
      it.s.len = __builtin_amdgcn_readlane(s.len, k);
      it.s.tiles = __builtin_amdgcn_readlane(s.tiles, k);
      it.s.span = __builtin_amdgcn_readlane(s.span, k);
      it.nsplit = __builtin_amdgcn_readlane(ns, k);
      const int local = w - before - (__builtin_amdgcn_readlane(incl, k) - __builtin_amdgcn_readlane(mine, k));
      const int sbase = slots + __builtin_amdgcn_readlane(sincl, k) - __builtin_amdgcn_readlane(states, k);
      const int at = by_tile ? local : (int)((uint32_t)local / (uint32_t)it.nsplit);
      it.split = by_tile ? 0 : local - at * it.nsplit;
      it.tile = it.s.tiles - 1 - at;  // the last tokens see the most rows: they go first
      it.slot = sbase + at * it.nsplit;
      return true;
    }
    before += __builtin_amdgcn_readlane(incl, 63);
    slots += __builtin_amdgcn_readlane(sincl, 63);
  }
  return false;
}

// row number of row j of a sequence's table (-1: not asked for, or a page id out of range)
__device__ inline int row_number(const PagedArgs& a, const int32_t* trow, int j, bool asked) {
  int id = -1;
  if (asked) {
    const uint32_t col = (uint32_t)j / (uint32_t)a.P;
    const int page = trow[col];
    if (page >= 0 && page < a.n_pages) id = page * a.P + (j - (int)col * a.P);
  }
  return id;
}

// States in the workspace, one slot per item of a split tile: (m, l) of its q rows and the scales of its values, then
// (all slots' apart) O^T in fp16, a power of two per lane and wave taken out, in the order of the accumulators.
template <class G>
__device__ inline float* state_f(const PagedArgs& a, int slot) {
  return (float*)(a.ws + kHeader) + (int64_t)slot * G::STATE_F;
}
template <class G>
__device__ inline uint8_t* state_o(const PagedArgs& a, int slot) {
  return a.ws + kHeader + (int64_t)a.slots * (G::STATE_F * 4) + (int64_t)slot * G::STATE_O;
}

// value wave vi (0 .. 4; wave kFirstValue + vi): first block and blocks
__device__ inline constexpr int units_of(int vi) { return vi == 0 ? 4 : 3; }
__device__ inline constexpr int first_unit(int vi) { return vi == 0 ? 0 : 1 + 3 * vi; }

// chunk ch (16 bytes) of output row r where the finished rows are staged (over the ring)
__device__ inline constexpr int out_at(int r, int ch) { return 1024 * r + 16 * (ch ^ (r & 15)); }

// What a workgroup works on, the same in all its waves.
struct Work {
  int slot;    // state slot, -1: the tile's only item
  int nh;      // q rows here
  int64_t row0;  // first of them in q and out
  int m0, p0, p_lo, p_hi;  // the first one's number in its sequence; positions of the sequence's first token, the tile's first and last
  int lo, nf;  // entry e < nf: row e; e >= nf: row lo + e - nf
  int e_begin, e_end, ntiles;
  bool once;  // the sequence's only tile: nobody else reads its rows in this call, but sequences that share its pages
};

// ---- row copies of one tile, dealt to the value waves (one instruction a row for columns 0..511, one per 8 rows for the
// rope tails, XOR-swizzled by row).  The row numbers are in registers by then (RowIds, read from the ring an
// iteration before), and a row's address is scalar: a copy costs its wave a few issue slots.
struct RowIds {
  int mine, tail;  // of row lane & 31; of the lane's row of this wave's tail copy
};
// the k-th copy of a tile (NB = 3: fp8 piece) that value wave vi takes (the wave with four blocks is dealt last)
__device__ inline constexpr int dealt(int vi, int k) { return kValueWaves - 1 - vi + kValueWaves * k; }
template <class G>
__device__ inline RowIds read_ids(const lds_i32_t* ids_s, int vi, int lane, int tl) {
  const lds_i32_t* id = ids_s + (tl % kIdTiles) * kTileRows;
  // copies 32 .. 35 are the tails': wave vi has number 32 + t, t = (dealt(vi, 0) - 32) mod 5, if that is below 4
  const int t = (dealt(vi, 0) + 3) % kValueWaves;
  return RowIds{max(id[lane & 31], 0), G::TAIL && t < 4 ? max(id[8 * t + (lane >> 3)], 0) : 0};
}
// 1 KB from a row at a scalar address, chunks swizzled (the s_nop as in dma16); nt: not kept in the L2
__device__ inline void copy_row(uint32_t lds_dst, uint64_t row, int x, int lane, bool nt) {
  const int at = 16 * (lane ^ row_swizzle(x));
  if (nt)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt" ::"s"(lds_dst), "v"(at), "s"(row) : "memory", "m0");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds_dst), "v"(at), "s"(row) : "memory", "m0");
}
// NT: past the caches, where no other tile of the sequence reads the rows (a decode step of 32 sequences 149 us against 156,
// 32 of 8192 rows 68 / 74, 256 of 8192 458 / 466; the 128-byte tails too: 151; rows that tiles share, a prompt's window:
// 210 against 200).  Sequences that share pages are not told apart, which costs little: 32 over one prefix of 8192 rows
// 57.8 / 57.2, 128 over 16384 311 / 308, 64 over 2048 with 300 rows each of their own 43.2 / 42.4; 8 over 8192 37.5 / 33.0.
template <class G, bool NT>
__device__ inline void issue_copies(const PagedArgs& a, uint32_t lds_base, const RowIds& id, int vi, int lane, int tl) {
  const uint32_t tbase = lds_base + (uint32_t)((tl % G::NBUF) * G::TILE_BYTES);
#pragma unroll
  for (int k = 0; k < (G::NDMA + kValueWaves - 1) / kValueWaves; k++) {
    const int x = dealt(vi, k);
    if (x < kTileRows) {
      const uint64_t row = (uint64_t)(uintptr_t)a.pages + (uint64_t)(uint32_t)__builtin_amdgcn_readlane(id.mine, x) * G::ROWB;
      copy_row(tbase + x * 1024, row, x, lane, NT);
    } else if (x < G::NDMA) {
      const int r0 = (x - kTileRows) * 8, r = r0 + (lane >> 3);
      dma16((const uint8_t*)a.pages + (int64_t)id.tail * G::ROWB + 1024 + 16 * ((lane & 7) ^ (r & 7)),
            __builtin_amdgcn_readfirstlane(tbase + G::MAIN_BYTES + r0 * 128));
    }
  }
}
template <class G>
__device__ inline void issue_tile(const PagedArgs& a, uint32_t lds_base, const RowIds& id, int vi, int lane, int tl, bool once) {
  // (at NB = 3 few sequences make one tile, and the choice alone costs a chunk 2 %)
  if (G::NB == 2 && once) issue_copies<G, true>(a, lds_base, id, vi, lane, tl);
  else issue_copies<G, false>(a, lds_base, id, vi, lane, tl);
}
// the same for 32 rows whose addresses `rowp` gives
template <class G, class F>
__device__ inline void copy_rows(uint32_t tbase, int vi, int lane, bool nt, F&& rowp) {
#pragma unroll
  for (int k = 0; k < (G::NDMA + kValueWaves - 1) / kValueWaves; k++) {
    const int x = dealt(vi, k);
    if (x < kTileRows) {
      copy_row(tbase + x * 1024, rowp(x), x, lane, nt);
    } else if (x < G::NDMA) {
      const int r0 = (x - kTileRows) * 8, r = r0 + (lane >> 3);
      dma16_nt((const uint8_t*)rowp(r) + 1024 + 16 * ((lane & 7) ^ (r & 7)),
               __builtin_amdgcn_readfirstlane(tbase + G::MAIN_BYTES + r0 * 128));
    }
  }
}

// ---- fp8 rows (e4m3 codes, one fp32 scale per 64 columns): a tile's codes in pieces of 16, 64 pieces at a time: main columns
// first, then the rope tails, so no wave instruction mixes the two.  At NB = 2 wave 2 has no q rows and takes most of
// them, the value waves kShare each; both keep two tiles' codes on their way (2 to 4 draft tokens of 64 sequences, 16 heads:
// 110 us; all pieces by the value waves 115, one tile ahead 121).  At NB = 3 the value waves share them.
constexpr int kShare = 2;
template <int D>
constexpr int kPieces8 = kTileRows * (D / 16) / 64;
template <int NB, int D>
constexpr int kMine8 = NB == 2 ? kShare : (kPieces8<D> + kValueWaves - 1) / kValueWaves;  // a value wave's
template <int K>
struct F8 {
  u32x4_t v[K];
  float s[K];
};
template <int D>
__device__ inline void f8_place(int x, int lane, int& r, int& cc) {
  if (x < 16) {
    r = 2 * x + (lane >> 5);
    cc = lane & 31;
  } else {
    r = (x - 16) * 16 + (lane >> 2);
    cc = 32 + (lane & 3);
  }
}
// pieces x0 + k step, k < K (of the last, those that exist)
template <int D, int K>
__device__ inline void f8_load(const PagedArgs& a, const lds_i32_t* ids_s, int x0, int step, int lane, int tl, F8<K>& f) {
  const lds_i32_t* id = ids_s + (tl % kIdTiles) * kTileRows;
#pragma unroll
  for (int k = K - 1; k >= 0; k--) {
    const int x = x0 + k * step;
    if (x < kPieces8<D>) {
      int r, cc;
      f8_place<D>(x, lane, r, cc);
      const int64_t row = max(id[r], 0);
      f.v[k] = *(const u32x4_t*)((const uint8_t*)a.pages + row * D + 16 * cc);
      f.s[k] = a.page_scales[row * (D / 64) + (cc >> 2)];
    }
  }
}
template <class G, int D, int K>
__device__ inline void f8_store(lds_u8_t* lds, int x0, int step, int lane, int tl, const F8<K>& f) {
  lds_u8_t* slot = lds + (tl % G::NBUF) * G::TILE_BYTES;
#pragma unroll
  for (int k = 0; k < K; k++) {
    const int x = x0 + k * step;
    if (x < kPieces8<D>) {
      int r, cc;
      f8_place<D>(x, lane, r, cc);
      uint32_t w[8];
      // a normal power-of-two scale: code x scale is a bf16 value, given exactly by the scaled
      // converter; any other scale: the fp32 product rounded to bf16
      const uint32_t su = __float_as_uint(f.s[k]);
      if ((su & 0x7fffffu) == 0 && su - 0x00800000u < 0x7f000000u) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
          w[2 * j] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(f.v[k][j], f.s[k], false));
          w[2 * j + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(f.v[k][j], f.s[k], true));
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const f32x2_t x0 = __builtin_amdgcn_cvt_pk_f32_fp8((int)f.v[k][j], false);
          const f32x2_t x1 = __builtin_amdgcn_cvt_pk_f32_fp8((int)f.v[k][j], true);
          w[2 * j] = pack_bf16x2(x0.x * f.s[k], x0.y * f.s[k]);
          w[2 * j + 1] = pack_bf16x2(x1.x * f.s[k], x1.y * f.s[k]);
        }
      }
      const u32x4_t w0 = {w[0], w[1], w[2], w[3]}, w1 = {w[4], w[5], w[6], w[7]};
      if (x < 16) {
        const int ch = (2 * cc) ^ row_swizzle(r);
        *(lds_u32x4_t*)(slot + r * 1024 + 16 * ch) = w0;
        *(lds_u32x4_t*)(slot + r * 1024 + 16 * (ch ^ 1)) = w1;
      } else {
        const int l0 = 2 * (cc - 32);
        *(lds_u32x4_t*)(slot + G::MAIN_BYTES + r * 128 + 16 * (l0 ^ (r & 7))) = w0;
        *(lds_u32x4_t*)(slot + G::MAIN_BYTES + r * 128 + 16 * ((l0 + 1) ^ (r & 7))) = w1;
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Score wave `wave` < NB: q rows 32 wave .. + 31, one to a lane pair (lanes r and r + 32 share q row r and the tile's rows in
// runs of four).  Iteration i multiplies tile i (D / 16 products of 32 rows x 32 q rows x 16, 32 cycles of the matrix
// pipe each) and, in the issue slots that the products leave, turns tile i - 1's scores to probabilities and writes
// them: nothing of the softmax but the look at its maximum, which fills the wait for the first K fragments, stands by itself.
// Scores are kept in base 2; a maximum further than e^8 above the reference moves the reference, everything else stays
// below e^8 of it.
template <class G, int D>
__device__ inline void score_role(const PagedArgs& a, const Work& w, const int32_t* trow, lds_u8_t* lds, int wave, int lane) {
  lds_i32_t* ids_s = (lds_i32_t*)(lds + G::IDS_OFF);
  lds_f32_t* al_s = (lds_f32_t*)(lds + G::AL_OFF);
  constexpr int STEPS = D / 16;
  const int h = lane >> 5, r = 32 * wave + (lane & 31);  // half, q row of the tile
  const bool idle = 32 * wave >= w.nh;  // no q rows: barriers (and row numbers) only
  constexpr float kLog2e = 1.44269504088896340736f;
  const float c2 = fabsf(a.scale) * kLog2e;
  const int rr = r < w.nh ? r : 0;  // (rows past nh are the tile's first)
  // entries that the q row sees: e < eh, and e < first or e >= past
  const int eh = max(w.p0 + (int)((uint32_t)(w.m0 + rr) / (uint32_t)a.H) + 1 - w.lo + w.nf, 0);
  const int past = a.window > 0 ? max(eh - a.window, 0) : 0;
  // entries below eh_all and outside [first, el_all) are seen by every q row of the tile
  const int eh_all = w.p_lo + 1 - w.lo + w.nf, el_all = a.window > 0 ? w.p_hi - a.window + 1 - w.lo + w.nf : 0;
  if (idle) {  // nothing to rescale, and no flags
    al_s[h * G::TILEQ + r] = 1.f;
    if (lane < 2) *(lds_i32_t*)(lds + G::FLAG_OFF + 16 * lane + 4 * wave) = 0;
  }
  // K of row lane & 31, step j: chunk 2 j + h of the main columns, 2 (j - 32) + h of the tail; the swizzle only turns bits,
  // so a step's address is step 0's xor 32 (j mod 8) (j mod 4 in the tail), and 256 (j / 8) on
  const uint32_t k_at = (uint32_t)(uintptr_t)lds + 1024 * (lane & 31) + 16 * (h ^ row_swizzle(lane & 31));
  const uint32_t t_at = (uint32_t)(uintptr_t)lds + G::MAIN_BYTES + 128 * (lane & 31) + 16 * (h ^ (lane & 7));
  auto ldk = [&](uint32_t buf, int j) -> u32x4_t {
    const uint32_t at = !G::TAIL || j < 32 ? ((buf + k_at) ^ (32 * (j & 7))) + 256 * (j >> 3) : (buf + t_at) ^ (32 * (j & 3));
    return *(const lds_u32x4_t*)(uintptr_t)at;
  };
  // Q^T of q row r, step j: elements 16 j + 8 h .. + 7, from the ring slot that its 32 q rows came to in a tile's layout; a
  // negative scale's sign goes into q
  bf16x8_t qf[STEPS];
#pragma unroll
  for (int j = 0; j < STEPS; j++) qf[j] = as_bf16x8(ldk((G::NBUF - G::NB + wave) * G::TILE_BYTES, j));
  if (a.scale < 0.f) {
#pragma unroll
    for (int j = 0; j < STEPS; j++) qf[j] = as_bf16x8(__builtin_bit_cast(u32x4_t, qf[j]) ^ 0x80008000u);
  }
  lds_barrier();  // Q's slots are free
  // the reference; below every score while there is none (exponentials of -inf against it are 0, and the first score seen
  // is past it)
  constexpr float kSlack = kRescaleSlack * kLog2e;
  float m_ref = -3e38f, l_lane = 0.f;
  // the row number of tile 7's entry lane & 31 as column and place in its page, and 32 rows' step
  int col = 0, off = 0, page = -1;
  const int step_col = (int)((uint32_t)kTileRows / (uint32_t)a.P), step_off = kTileRows - step_col * a.P;
  if (wave == 0) {
    const int e = w.e_begin + (kIdTiles - 1) * kTileRows + (lane & 31), j = e < w.nf ? e : w.lo + (e - w.nf);
    col = (int)((uint32_t)j / (uint32_t)a.P);
    off = j - col * a.P;
    if (e < w.e_end) page = trow[col];
  }
  // page: of tile i + 6's entry, read in iteration i - 1 and used in iteration i, so that nothing waits for it
  auto row_numbers = [&](int i) {
    if (wave != 0) return;
    // tile i + 6's to the slot of tile i - 2, which nobody masks by any more (both halves of the wave alike)
    if (i + 6 < w.ntiles)
      ids_s[((i + 6) % kIdTiles) * kTileRows + (lane & 31)] = (uint32_t)page < (uint32_t)a.n_pages ? page * a.P + off : -1;
    if (i + 7 < w.ntiles) {
      const int e = w.e_begin + (i + 7) * kTileRows + (lane & 31);
      // rows follow each other by 32, but where the first rows end
      off += step_off;
      col += step_col;
      if (off >= a.P) {
        off -= a.P;
        col++;
      }
      if (w.nf > 0 && w.e_begin + (i + 6) * kTileRows < w.nf) {
        const int j = e < w.nf ? e : w.lo + (e - w.nf);
        col = (int)((uint32_t)j / (uint32_t)a.P);
        off = j - col * a.P;
      }
      page = -1;
      if (e < w.e_end) page = trow[col];
    }
  };
  // scores of a tile of which some q row does not see some row: scaled, -inf there; whether one, seen or not, is not finite
  // (0 x it is not 0).  The rows that the q row sees as bits: those whose row number is there (a ballot), below eh, and
  // from `past` on or below first; then per score a bit spread to a word, and bitwise selects.
  auto mask = [&](f32x16_t& s, int i) -> bool {
    const int e0 = w.e_begin + i * kTileRows;
    const uint32_t there = (uint32_t)__builtin_amdgcn_ballot_w64(ids_s[(i % kIdTiles) * kTileRows + (lane & 31)] >= 0);
    auto below = [](int n) -> uint32_t { return n >= 32 ? 0xffffffffu : (1u << max(n, 0)) - 1; };  // the bits below n
    const uint32_t mine = (there & below(eh - e0) & (~below(past - e0) | below(a.first - e0))) >> (4 * h);
    float z = 0.f;
#pragma unroll
    for (int k = 0; k < 16; k++) {
      const uint32_t m = (uint32_t)__builtin_amdgcn_sbfe((int)mine, 8 * (k >> 2) + (k & 3), 1);
      z = __builtin_fmaf(s[k], 0.f, z);
      s[k] = __uint_as_float((__float_as_uint(s[k] * c2) & m) | (__float_as_uint(-SMLA_INF) & ~m));
    }
    return !(z == 0.f);
  };
  // whether every q row of the tile sees every row of tile i (its row numbers v are all there)
  auto is_open = [&](int i, const i32x4_t& v) -> bool {
    const int e0 = w.e_begin + i * kTileRows;
    return e0 + kTileRows <= eh_all && (e0 >= el_all || e0 + kTileRows <= a.first) &&
           __builtin_amdgcn_ballot_w64(min(min(v[0], v[1]), min(v[2], v[3])) < 0) == 0;
  };
  auto ids_of = [&](int i) { return *(const lds_i32x4_t*)(ids_s + (i % kIdTiles) * kTileRows + 4 * (lane & 7)); };
  constexpr int PF = G::TAIL ? 5 : 4;  // fragments read ahead (more only crowd the LDS at a tile's start)
  u32x4_t kf[PF];
  // the products of tile i; `between` j runs after step j's
  auto products = [&](f32x16_t& s, int i, auto&& before, auto&& between) {
    const uint32_t buf = (uint32_t)((i % G::NBUF) * G::TILE_BYTES);
#pragma unroll
    for (int j = 0; j < PF; j++) kf[j] = ldk(buf, j);
#pragma unroll
    for (int k = 0; k < 16; k++) s[k] = 0.f;
    __builtin_amdgcn_sched_barrier(0);
    before();
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < STEPS; j++) {
      const bf16x8_t k = as_bf16x8(kf[j % PF]);
      if (j + PF < STEPS) kf[j % PF] = ldk(buf, j + PF);
      s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k, qf[j], s, 0, 0, 0);
      between(j);
      __builtin_amdgcn_sched_barrier(0);  // keep the reads PF steps ahead of their products
    }
  };
  bool open = false;
  // Iteration i: tile i's products into `now`, tile i - 1's scores `old` to P.
  auto iteration = [&](int i, f32x16_t& now, f32x16_t& old) {
    const bool more = i < w.ntiles;
    const float cm = open ? c2 : 1.f;  // what turns tile i - 1's scores to base 2 (1: masked, and scaled, already)
    float alpha = 1.f;                 // e^(old - new reference)
    bool odd = false;
    const bool masked = !open;
    if (masked) odd = mask(old, i - 1);
    float least = 0.f;  // of the scores; -inf where a seen row counts for nothing (masked: known already)
    auto look = [&]() {  // the reference moves to the tile's maximum where that is past it
      float x = fmaxf(old[0], old[1]);
#pragma unroll
      for (int k = 2; k < 16; k += 2) x = fmaxf(fmaxf(x, old[k]), old[k + 1]);
      x *= cm;
      if (__builtin_amdgcn_ballot_w64(x > m_ref + kSlack)) {
        const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = fmaxf(__uint_as_float(y[0]), __uint_as_float(y[1]));
        if (x > m_ref + kSlack) {
          alpha = __builtin_amdgcn_exp2f(m_ref - x);
          l_lane *= alpha;
          m_ref = x;
        }
      }
    };
    auto expo = [&](int k) {
      if ((k & 1) == 0) least = fminf(fminf(least, old[k]), old[k + 1]);
      old[k] = __builtin_amdgcn_exp2f(old[k] * cm - m_ref);
    };
    auto put = [&](int q) {
      l_lane += (old[4 * q] + old[4 * q + 1]) + (old[4 * q + 2] + old[4 * q + 3]);
      *(lds_u32x2_t*)(lds + G::P_OFF + ((i - 1) & 1) * G::PBUF + p_at(r, q) + 8 * h) =
          u32x2_t{pack2(old[4 * q], old[4 * q + 1]), pack2(old[4 * q + 2], old[4 * q + 3])};
    };
    auto put_alpha = [&]() {
      al_s[((i - 1) & 1) * G::TILEQ + r] = alpha;
      const uint64_t any = __builtin_amdgcn_ballot_w64(odd | (!masked & (least == -SMLA_INF)));
      if (lane == 0) *(lds_i32_t*)(lds + G::FLAG_OFF + 16 * ((i - 1) & 1) + 4 * wave) = any != 0;
    };
    if (more) {
      i32x4_t v;
      bool next = false;
      products(now, i, look, [&](int j) {
        if (j < 16) expo(j);
        if (j >= 16 && j < 24 && (j & 1) == 0) put((j - 16) / 2);
        if (j == 24) put_alpha();
        if (j == 25) v = ids_of(i);
        if (j == 26) row_numbers(i);
        if (j == 29) next = is_open(i, v);
      });
      open = next;
    } else {
      look();
#pragma unroll
      for (int k = 0; k < 16; k++) expo(k);
#pragma unroll
      for (int q = 0; q < 4; q++) put(q);
      put_alpha();
    }
  };
  // the compiler's own count: no load is in flight from here on but row_numbers' one, so the loop waits for none
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
  f32x16_t s0, s1;
  if (!idle && w.ntiles > 0) {
    open = is_open(0, ids_of(0));
    products(s0, 0, [] {}, [](int) {});
  }
  lds_barrier();
  for (int i = 1; i <= w.ntiles; i += 2) {
    if (!idle) iteration(i, s1, s0);
    lds_barrier();
    if (i + 1 > w.ntiles) break;
    if (!idle) iteration(i + 1, s0, s1);
    lds_barrier();
  }
  lds_barrier();  // (the value waves' last tile)
  // (m, l): for the value waves' final scaling, or the state's
  const float l = l_lane + __shfl_xor(l_lane, 32, 64);
  if (h == 0) {
    if (w.slot >= 0) *(f32x2_t*)(state_f<G>(a, w.slot) + 2 * r) = f32x2_t{m_ref, l};
    al_s[2 * r] = m_ref;
    al_s[2 * r + 1] = l;
  }
  lds_barrier();
}

// ---------------------------------------------------------------------------------------------
// Value wave vi with NU blocks of 32 columns from block u0 on.
template <class G, int D, bool FP8, int NU>
__device__ inline void value_role(const PagedArgs& a, const Work& w, lds_u8_t* lds, int vi, int u0, int lane) {
  constexpr int NB = G::NB;
  const lds_i32_t* ids_s = (const lds_i32_t*)(lds + G::IDS_OFF);
  const lds_f32_t* al_s = (const lds_f32_t*)(lds + G::AL_OFF);
  const uint32_t lds_base = (uint32_t)(uintptr_t)lds;
  const int nb = (w.nh + 31) / 32;  // blocks of q rows in use (the others' products are not stored)
  const int my_dma = (G::NDMA - dealt(vi, 0) + kValueWaves - 1) / kValueWaves;
  RowIds ids{0, 0};  // of the next tile to request
  f32x16_t o[NU][NB];
#pragma unroll
  for (int u = 0; u < NU; u++)
#pragma unroll
    for (int n = 0; n < NB; n++)
#pragma unroll
      for (int r = 0; r < 16; r++) o[u][n][r] = 0.f;
  // V^T provider address inside a 16-row step: group j = lane >> 4 covers value columns 16 (j & 1) .. of a block and
  // rows 8 (j >> 1) ..; lane J = lane & 15 supplies row J >> 2, columns 4 (J & 3) .. + 3.  Of a block's chunk the swizzle
  // turns the number in its group of four (alike in all blocks) and, by the row's two low bits, the block's place
  // among four
  const int vj = lane >> 4, vJ = lane & 15;
  const int tr_row = 8 * (vj >> 1) + (vJ >> 2), tr_ch = 2 * (vj & 1) + ((vJ & 3) >> 1);
  const int tr_lo = 1024 * tr_row + 16 * (tr_ch ^ (row_swizzle(tr_row) & 3)) + 8 * (vJ & 1);  // rows vJ >> 2 of each eight
  const int tr_hi = 1024 * (tr_row + 4) + 16 * (tr_ch ^ (row_swizzle(tr_row + 4) & 3)) + 8 * (vJ & 1);  // 4 + (vJ >> 2)
  const int tr_turn = 64 * (vJ >> 2);
  int pr[2];  // chunk 2 ks + (lane >> 5) of q row lane & 31 (+ 32 n)
#pragma unroll
  for (int ks = 0; ks < 2; ks++) pr[ks] = p_at(lane & 31, 2 * ks + (lane >> 5));
  // fp8 codes on their way: of one tile, of two where registers are left
  constexpr bool DEEP = FP8 && NB == 2;
  F8<kMine8<NB, D>> f8, f8_next;
  const int x0 = DEEP ? vi : dealt(vi, 0);
  __builtin_assume(x0 >= 0 && x0 < kValueWaves);
  const int last = max(w.ntiles - 1, 0);
  // ---- Q rows to the last NB ring slots in a tile's layout (read once: not kept in the L2, unless the tile is split), then
  // the tiles that the other slots hold (fp8: tile 0, and the next ones' codes)
  constexpr int EARLY = G::NBUF - NB;
  auto request_q = [&](bool nt) {
#pragma unroll
    for (int n = 0; n < NB; n++)
      if (32 * n < w.nh)
        copy_rows<G>(lds_base + (EARLY + n) * G::TILE_BYTES, vi, lane, nt, [&](int x) {
          return (uint64_t)(uintptr_t)a.q + (uint64_t)(w.row0 + (32 * n + x < w.nh ? 32 * n + x : 0)) * G::ROWB;
        });
  };
  if (w.slot < 0) request_q(true);
  else request_q(false);
  lds_barrier();  // the first row numbers are there
  if constexpr (FP8) {
    // (past the last tile: the last once more, so that the loads in flight are counted alike on all paths)
    f8_load<D>(a, ids_s, x0, kValueWaves, lane, 0, f8);
    f8_store<G, D>(lds, x0, kValueWaves, lane, 0, f8);
    f8_load<D>(a, ids_s, x0, kValueWaves, lane, min(1, last), f8);
    if constexpr (DEEP) f8_load<D>(a, ids_s, x0, kValueWaves, lane, min(2, last), f8_next);
  } else {
    for (int tl = 0; tl < min(w.ntiles, EARLY); tl++)
      issue_tile<G>(a, lds_base, read_ids<G>(ids_s, vi, lane, tl), vi, lane, tl, w.once);
  }
  // Q and tile 0 are there
  if (FP8 || w.ntiles <= 1) {
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0), in the compiler's own count too
    asm volatile("" ::: "memory");
  } else {
    wait_vm((EARLY - 1) * my_dma);
  }
  lds_barrier();
  lds_barrier();  // the score waves have read Q
  if constexpr (!FP8) {
    for (int tl = EARLY; tl < min(w.ntiles, G::NBUF); tl++)
      issue_tile<G>(a, lds_base, read_ids<G>(ids_s, vi, lane, tl), vi, lane, tl, w.once);
    if (G::NBUF < w.ntiles) ids = read_ids<G>(ids_s, vi, lane, G::NBUF);
  }
  // Iteration i: the score waves finish tile i - 1 and begin tile i, tile i - 2 is consumed here, and tile i + 1 goes
  // to the slot of tile i - 3, to be there at the iteration's end.
  auto iteration = [&](int i, F8<kMine8<NB, D>>& f) {
    if constexpr (FP8) {
      if (i + 1 < w.ntiles) f8_store<G, D>(lds, x0, kValueWaves, lane, i + 1, f);
      f8_load<D>(a, ids_s, x0, kValueWaves, lane, min(i + 2 + DEEP, last), f);
    } else {
      if (i >= 3 && i + 1 < w.ntiles) {
        issue_tile<G>(a, lds_base, ids, vi, lane, i + 1, w.once);
        if (i + 2 < w.ntiles) ids = read_ids<G>(ids_s, vi, lane, i + 2);
      }
    }
    if (i >= 2) {
      const int tp = i - 2;  // its P was written in the last iteration
      lds_u8_t* buf = lds + (tp % G::NBUF) * G::TILE_BYTES;
      const lds_u8_t* pbuf = lds + G::P_OFF + (tp & 1) * G::PBUF;
      // step st: rows 16 (st / NU) .. + 15, block st % NU; V^T is read AHEAD steps early
      constexpr int AHEAD = NU * NB < 12 ? 2 : 1;  // (192 accumulators leave room for one)
      const lds_u8_t *vlo = buf + tr_lo, *vhi = buf + tr_hi;
      auto ldv = [&](int st) -> u32x4_t {
        const int u = u0 + st % NU, at = 16 * 1024 * (st / NU), block = ((64 * (u & 3)) ^ tr_turn) + 256 * (u >> 2);
        const v4i16_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_t*)(vlo + block + at));
        const v4i16_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_t*)(vhi + block + at));
        return __builtin_bit_cast(u32x4_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
      };
      auto ldp = [&](int ks, int n) { return as_bf16x8(*(const lds_u32x4_t*)(pbuf + pr[ks] + 32 * 64 * n)); };
      float al[NB];
#pragma unroll
      for (int n = 0; n < NB; n++) al[n] = al_s[(tp & 1) * G::TILEQ + 32 * n + (lane & 31)];
      const i32x4_t flag = *(const lds_i32x4_t*)(lds + G::FLAG_OFF + 16 * (tp & 1));
      bf16x8_t pf[NB];
      u32x4_t va[AHEAD + 1];
#pragma unroll
      for (int n = 0; n < NB; n++) pf[n] = ldp(0, n);
#pragma unroll
      for (int st = 0; st < AHEAD; st++) va[st] = ldv(st);
      __builtin_amdgcn_sched_barrier(0);
      bool turn = false;
#pragma unroll
      for (int n = 0; n < NB; n++) turn |= al[n] != 1.f;
      if (__builtin_amdgcn_ballot_w64(turn)) {
#pragma unroll
        for (int n = 0; n < NB; n++)
#pragma unroll
          for (int u = 0; u < NU; u++) o[u][n] *= al[n];
      }
      int odd = flag[0];
#pragma unroll
      for (int n = 1; n < NB; n++) odd |= flag[n];
      if (__builtin_amdgcn_readfirstlane(odd)) {
        // this wave's columns (nobody else reads them by now): 4 NU chunks of each of 32 rows
        for (int x = lane; x < kTileRows * 4 * NU; x += 64) {
          const int row = x / (4 * NU), ch = 4 * u0 + x - row * (4 * NU);
          lds_u32x4_t* at = (lds_u32x4_t*)(buf + row * 1024 + 16 * (ch ^ row_swizzle(row)));
          u32x4_t y = *at;
#pragma unroll
          for (int k = 0; k < 4; k++) y[k] = finite2(y[k]);
          *at = y;
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
        for (int st = 0; st < AHEAD; st++) va[st] = ldv(st);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int st = 0; st < 2 * NU; st++) {
        const bf16x8_t v = as_bf16x8(va[st % (AHEAD + 1)]);
        if (st + AHEAD < 2 * NU) va[(st + AHEAD) % (AHEAD + 1)] = ldv(st + AHEAD);
#pragma unroll
        for (int n = 0; n < NB; n++) {
          o[st % NU][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, pf[n], o[st % NU][n], 0, 0, 0);
          if (st == NU - 1) pf[n] = ldp(1, n);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if constexpr (!FP8) {
      // tile i + 1 has landed (the newest requested: 3 at first, then i + 1)
      if (i >= 2) wait_vm(0);
      else if (i + 1 < w.ntiles) wait_vm(max(0, min(3, w.ntiles - 1) - (i + 1)) * my_dma);
    }
    lds_barrier();
  };
  if constexpr (DEEP) {
    // in pairs, each register set with its own half (a way out between the halves would make the compiler wait for all
    // loads); of an odd number the first, which has no products, by itself
    int i = w.ntiles & 1;
    if (i) {
      if (w.ntiles > 1) f8_store<G, D>(lds, x0, kValueWaves, lane, 1, f8);
      f8 = f8_next;
      f8_load<D>(a, ids_s, x0, kValueWaves, lane, min(3, last), f8_next);
      lds_barrier();
    }
    for (; i <= w.ntiles; i += 2) {
      iteration(i, f8);
      iteration(i + 1, f8_next);
    }
  } else {
    for (int i = 0; i <= w.ntiles + 1; i++) iteration(i, f8);
  }
  lds_barrier();  // (m, l) in LDS
#pragma unroll
  for (int n = 0; n < NB; n++) {
    if (n >= nb) continue;
    const int r = 32 * n + (lane & 31);
    // O^T of block u: register k holds column 8 (k >> 2) + 4 (lane >> 5) + (k & 3) of q row r; one lane swap per
    // pair of packed registers gives each lane 8 columns in a row, 16 h + 8 (lane >> 5) .. + 7
    if (w.slot >= 0) {
      // the largest magnitude of the lane pair's 32 NU columns sets their scale: fp16 keeps 11 bits of those down to 2^-14 of it
      float top = 0.f;
#pragma unroll
      for (int u = 0; u < NU; u++)
#pragma unroll
        for (int k = 0; k < 16; k++) top = fmaxf(top, fabsf(o[u][n][k]));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const uint32_t e = min(max(__float_as_uint(top) >> 23, 1u), 253u);  // 2^(e-127) <= top < 2^(e-126)
      const float inv = __uint_as_float((254u - e) << 23);
      state_f<G>(a, w.slot)[2 * G::TILEQ + (vi * NB + n) * 64 + lane] = __uint_as_float(e << 23);
      uint8_t* blk = state_o<G>(a, w.slot) + (u0 * NB + n) * 2048 + 16 * lane;
#pragma unroll
      for (int u = 0; u < NU; u++) {
        uint32_t d[8];
#pragma unroll
        for (int k = 0; k < 8; k++)
          d[k] = __builtin_bit_cast(uint32_t, f16x2_t{(_Float16)(o[u][n][2 * k] * inv), (_Float16)(o[u][n][2 * k + 1] * inv)});
#pragma unroll
        for (int k = 0; k < 8; k += 4) {
          const auto x0 = __builtin_amdgcn_permlane32_swap(d[k], d[k + 2], false, false);
          const auto x1 = __builtin_amdgcn_permlane32_swap(d[k + 1], d[k + 3], false, false);
          __builtin_nontemporal_store(u32x4_t{x0[0], x1[0], x0[1], x1[1]}, (u32x4_t*)(blk + u * NB * 2048 + (k >> 2) * 1024));
        }
      }
    } else {
      const float M = al_s[2 * r], L = al_s[2 * r + 1];
      float inv = 0.f;  // no row seen: 0
      if (!(L == 0.f)) {
        const float snk = a.sink && r < w.nh ? a.sink[(uint32_t)(w.m0 + r) % (uint32_t)a.H] : -SMLA_INF;
        inv = 1.0f / (L + (snk == -SMLA_INF ? 0.f : __builtin_amdgcn_exp2f(snk * 1.44269504088896340736f - M)));
      }
#pragma unroll
      for (int u = 0; u < NU; u++) {
        uint32_t d[8];
#pragma unroll
        for (int k = 0; k < 8; k++) d[k] = pack2(o[u][n][2 * k] * inv, o[u][n][2 * k + 1] * inv);
#pragma unroll
        for (int k = 0; k < 8; k += 4) {
          const auto x0 = __builtin_amdgcn_permlane32_swap(d[k], d[k + 2], false, false);
          const auto x1 = __builtin_amdgcn_permlane32_swap(d[k + 1], d[k + 3], false, false);
          *(lds_u32x4_t*)(lds + out_at(r, 4 * (u0 + u) + (k >> 1) + (lane >> 5))) = u32x4_t{x0[0], x1[0], x0[1], x1[1]};
        }
      }
    }
  }
}

// Wave 2 at NB = 2 over fp8 pages: the pieces that the value waves leave, requested two tiles ahead; it keeps their barriers.
template <class G, int D>
__device__ inline void feed_role(const PagedArgs& a, const Work& w, lds_u8_t* lds, int lane) {
  constexpr int X0 = kShare * kValueWaves, K = kPieces8<D> - X0;
  const lds_i32_t* ids_s = (const lds_i32_t*)(lds + G::IDS_OFF);
  const int last = max(w.ntiles - 1, 0);
  F8<K> f8, f8_next;
  f8_load<D>(a, ids_s, X0, 1, lane, 0, f8);
  f8_store<G, D>(lds, X0, 1, lane, 0, f8);
  f8_load<D>(a, ids_s, X0, 1, lane, min(1, last), f8);
  f8_load<D>(a, ids_s, X0, 1, lane, min(2, last), f8_next);
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
  lds_barrier();
  lds_barrier();
  auto iteration = [&](int i, F8<K>& f) {
    if (i + 1 < w.ntiles) f8_store<G, D>(lds, X0, 1, lane, i + 1, f);
    f8_load<D>(a, ids_s, X0, 1, lane, min(i + 3, last), f);
    __builtin_amdgcn_sched_barrier(0);
    lds_barrier();
  };
  int i = w.ntiles & 1;  // (pairs: as in value_role)
  if (i) {
    if (w.ntiles > 1) f8_store<G, D>(lds, X0, 1, lane, 1, f8);
    f8 = f8_next;
    f8_load<D>(a, ids_s, X0, 1, lane, min(3, last), f8_next);
    lds_barrier();
  }
  for (; i <= w.ntiles; i += 2) {
    iteration(i, f8);
    iteration(i + 1, f8_next);
  }
  lds_barrier();
}

template <int D, int NB, bool FP8>
__global__ __launch_bounds__(64 * kWaves) void paged_attn_kernel(const PagedArgs a) {
  using G = GeoP<D, NB>;
  extern __shared__ __align__(256) uint8_t lds_generic[];
  lds_u8_t* lds = (lds_u8_t*)lds_generic;
  lds_i32_t* ids_s = (lds_i32_t*)(lds + G::IDS_OFF);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  Item it;
  int rps;
  {
    const Seq s0 = load_seq<G::TILEQ>(a, lane);
    rps = plan_rps<G::TILEQ>(a, s0, lane);
    if (blockIdx.x == 0 && tid == 0) *(int*)a.ws = rps;
    if (!find_item<G::TILEQ>(a, s0, lane, rps, blockIdx.x, false, it)) return;
  }
  if (it.nsplit > 1 && it.slot + it.nsplit > a.slots) return;  // lengths that no batch of T tokens has
  Work w;
  const int rows_b = it.s.n * a.H;
  w.m0 = it.tile * G::TILEQ;
  w.once = it.s.tiles == 1;
  w.slot = it.nsplit > 1 ? it.slot + it.split : -1;
  w.nh = min(G::TILEQ, rows_b - w.m0);
  w.row0 = (int64_t)it.s.beg * a.H + w.m0;
  w.p0 = it.s.len - it.s.n;
  w.p_lo = w.p0 + (int)((uint32_t)w.m0 / (uint32_t)a.H);
  w.p_hi = w.p0 + (int)((uint32_t)(w.m0 + w.nh - 1) / (uint32_t)a.H);
  const int w_lo = w.p_lo - a.window + 1;
  w.lo = a.window > 0 && w_lo > 0 ? w_lo : 0;
  const int64_t cap = (int64_t)a.cols * a.P;  // rows from it on are not in the table, nor are first rows
  const int top = (int)min((int64_t)w.p_hi + 1, cap);  // rows below it
  w.nf = (int)min((int64_t)min(a.first, w.lo), cap);
  const int entries = w.nf + max(0, top - w.lo);  // (the window may start past the table: its first rows are seen still)
  const int part = ceil_div(ceil_div(it.s.span, it.nsplit), kTileRows) * kTileRows;
  w.e_begin = (int)min((int64_t)it.split * part, (int64_t)entries);
  w.e_end = min(entries, w.e_begin + part);
  w.ntiles = w.e_end > w.e_begin ? (w.e_end - w.e_begin + kTileRows - 1) / kTileRows : 0;
  const int32_t* trow = a.table + it.b * a.ld_table;
  if (wave < kFirstValue) {
    // the first eight tiles' row numbers: six, then (wave 0) two, there at the next barrier
    auto first_numbers = [&](int x) {
      const int e = w.e_begin + x;
      ids_s[x] = row_number(a, trow, e < w.nf ? e : w.lo + (e - w.nf), e < w.e_end);
    };
    first_numbers(tid);
    lds_barrier();
    if (tid < kIdTiles * kTileRows - 64 * kFirstValue) first_numbers(tid + 64 * kFirstValue);
    if (wave < NB) {
      lds_barrier();  // Q and tile 0 have landed
      score_role<G, D>(a, w, trow, lds, wave, lane);
    } else if constexpr (FP8 && NB == 2) {
      feed_role<G, D>(a, w, lds, lane);
    } else {
      for (int i = 0; i < w.ntiles + 5; i++) lds_barrier();
    }
  } else if (wave == kFirstValue) {
    value_role<G, D, FP8, units_of(0)>(a, w, lds, 0, first_unit(0), lane);
  } else {
    value_role<G, D, FP8, units_of(1)>(a, w, lds, wave - kFirstValue, first_unit(wave - kFirstValue), lane);
  }
  if (w.slot >= 0) return;
  lds_barrier();  // the rows are staged
  // the tile's q rows are consecutive rows of out, a kilobyte each; nothing here reads them again
  uint8_t* dst = (uint8_t*)(a.out + w.row0 * 512) + 16 * lane;
  for (int r = wave; r < w.nh; r += kWaves)
    __builtin_nontemporal_store(*(const lds_u32x4_t*)(lds + out_at(r, lane)), (u32x4_t*)(dst + (int64_t)r * 1024));
}

// ---------------------------------------------------------------------------------------------
// Joins the states of split tiles, in pieces of 1 KB (8 values of 32 q rows, twice).  A workgroup takes GROUP pieces of a tile
// at a time.  One piece by all its waves: wave w the splits w, w + WAVES, .. with a running maximum, the waves' sums then
// through LDS in a fixed order (kFewWaves: one tile of 65 splits 5.5 us, with four waves 6.5, with 16 8.3).
// Where there are pieces enough (GROUP 4, four waves) and a tile has at most kAlone splits,
// a piece a wave, which needs no LDS and no barriers: 1366 tiles of 2 or 3 splits 106 us against 254 (4.2 TB/s), 64 tiles of
// 3 to 6 8.5 against 13.9, 32 tiles of 8 9.6 against 12.9.
// Workgroups walk the pieces of all split tiles; with `fill` they also clear the tokens of no sequence.
constexpr int kFewWaves = 8, kMergeBatch = 8, kAlone = 16;

template <int D, int NB, int GROUP, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void paged_merge_kernel(const PagedArgs a) {
  using G = GeoP<D, NB>;
  constexpr int kPieces = kUnits * NB * 2;
  __shared__ float red[WAVES][64][10];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const Seq s0 = load_seq<G::TILEQ>(a, lane);
  const int rps = __builtin_amdgcn_readfirstlane(*(const int*)a.ws);
  constexpr uint32_t kGroups = kPieces / GROUP;
  for (uint32_t x = blockIdx.x;; x += gridDim.x) {
    Item it;
    const uint32_t tile = x / kGroups, piece0 = (x - tile * kGroups) * GROUP;
    if (!find_item<G::TILEQ>(a, s0, lane, rps, (int)tile, true, it)) break;
    if (it.slot + it.nsplit > a.slots) continue;
    const int m0 = it.tile * G::TILEQ, rows_b = it.s.n * a.H;
    // the splits from, from + step, .. of a piece: maximum, sum, values
    struct Sum {
      float m, l, acc[8];
    };
    auto gather = [&](int piece, int from, int step) -> Sum {
      const int u = piece / (2 * NB), n = (piece >> 1) % NB, vi = u < 4 ? 0 : (u - 1) / 3, row = 32 * n + (lane & 31);
      Sum t;
      t.m = -SMLA_INF;
      t.l = 0.f;
#pragma unroll
      for (int k = 0; k < 8; k++) t.acc[k] = 0.f;
      for (int sp0 = from; sp0 < it.nsplit; sp0 += step * kMergeBatch) {
        f32x2_t ml[kMergeBatch];
        float sc[kMergeBatch];
        u32x4_t v[kMergeBatch];
#pragma unroll
        for (int k = 0; k < kMergeBatch; k++) {
          const int sp = sp0 + step * k;
          if (sp < it.nsplit) {
            const float* f = state_f<G>(a, it.slot + sp);
            ml[k] = *(const f32x2_t*)(f + 2 * row);
            sc[k] = f[2 * G::TILEQ + (vi * NB + n) * 64 + lane];
            v[k] = *(const u32x4_t*)(state_o<G>(a, it.slot + sp) + piece * 1024 + 16 * lane);
          }
        }
        float top = t.m;
#pragma unroll
        for (int k = 0; k < kMergeBatch; k++)
          if (sp0 + step * k < it.nsplit) top = fmaxf(top, ml[k][0]);
        const float keep = t.m > -SMLA_INF ? __builtin_amdgcn_exp2f(t.m - top) : (top == t.m ? 1.f : 0.f);
        t.l *= keep;
#pragma unroll
        for (int j = 0; j < 8; j++) t.acc[j] *= keep;
        t.m = top;
#pragma unroll
        for (int k = 0; k < kMergeBatch; k++)
          if (sp0 + step * k < it.nsplit) {
            // a state without a maximum has l = 0 (nothing seen) or NaN
            const float e = ml[k][0] > -SMLA_INF ? __builtin_amdgcn_exp2f(ml[k][0] - t.m) : 1.f;
            t.l += ml[k][1] * e;
            const float es = e * sc[k];
#pragma unroll
            for (int j = 0; j < 4; j++) {
              const uint32_t word = v[k][j];  // (a bit cast of a vector's element itself takes element 0)
              const f16x2_t h2 = __builtin_bit_cast(f16x2_t, word);
              t.acc[2 * j] += (float)h2[0] * es;
              t.acc[2 * j + 1] += (float)h2[1] * es;
            }
          }
      }
      return t;
    };
    auto finish = [&](int piece, const Sum& t) {
      const int u = piece / (2 * NB), n = (piece >> 1) % NB, half = piece & 1, row = 32 * n + (lane & 31);
      if (m0 + row >= rows_b) return;
      float inv = 0.f;
      if (!(t.l == 0.f)) {
        const float snk = a.sink ? a.sink[(uint32_t)(m0 + row) % (uint32_t)a.H] : -SMLA_INF;
        inv = 1.0f / (t.l + (snk == -SMLA_INF ? 0.f : __builtin_amdgcn_exp2f(snk * 1.44269504088896340736f - t.m)));
      }
      u32x4_t o;
#pragma unroll
      for (int j = 0; j < 4; j++) o[j] = pack2(t.acc[2 * j] * inv, t.acc[2 * j + 1] * inv);
      *(u32x4_t*)(a.out + ((int64_t)it.s.beg * a.H + m0 + row) * 512 + 32 * u + 16 * half + 8 * (lane >> 5)) = o;
    };
    if constexpr (GROUP > 1)
      if (it.nsplit <= kAlone) {
        finish((int)piece0 + wave, gather((int)piece0 + wave, 0, 1));
        continue;
      }
    for (int piece = (int)piece0; piece < (int)piece0 + GROUP; piece++) {
      const Sum t = gather(piece, wave, WAVES);
      __syncthreads();  // the last piece's sums are read
      red[wave][lane][0] = t.m;
      red[wave][lane][1] = t.l;
#pragma unroll
      for (int j = 0; j < 8; j++) red[wave][lane][2 + j] = t.acc[j];
      __syncthreads();
      if (wave == 0) {
        Sum y;
        y.m = t.m;
#pragma unroll
        for (int k = 1; k < WAVES; k++) y.m = fmaxf(y.m, red[k][lane][0]);
        y.l = 0.f;
#pragma unroll
        for (int j = 0; j < 8; j++) y.acc[j] = 0.f;
#pragma unroll
        for (int k = 0; k < WAVES; k++) {
          const float mk = red[k][lane][0], e = mk > -SMLA_INF ? __builtin_amdgcn_exp2f(mk - y.m) : 1.f;
          y.l += red[k][lane][1] * e;
#pragma unroll
          for (int j = 0; j < 8; j++) y.acc[j] += red[k][lane][2 + j] * e;
        }
        finish(piece, y);
      }
    }
  }
  if (a.fill) {
    // 16-byte pieces of the tokens before the first sequence and behind the last
    const int64_t tok = (int64_t)a.H * 64, to = a.T * tok, first = min(max(a.cu[0], 0), a.T) * tok;
    const int64_t gap = max(min(max(a.cu[a.B], 0), a.T) * tok - first, (int64_t)0);
    const int64_t at = (int64_t)blockIdx.x * blockDim.x + threadIdx.x, step = (int64_t)gridDim.x * blockDim.x;
    for (int64_t i = at; i < to - gap; i += step) *(u32x4_t*)(a.out + (i < first ? i : i + gap) * 8) = u32x4_t{0u, 0u, 0u, 0u};
    // and of the sequences that were not granted theirs
    for (int b0 = 0; a.granted && b0 < a.B; b0 += 64) {
      const int b = b0 + lane;
      int c0 = 0, c1 = 0;
      if (b < a.B && a.granted[b] == 0) {
        c0 = min(max(a.cu[b], 0), a.T);
        c1 = min(max(a.cu[b + 1], 0), a.T);
      }
      for (uint64_t left = __builtin_amdgcn_ballot_w64(c0 < c1); left; left &= left - 1) {
        const int k = (int)__builtin_ctzll(left);
        const int64_t end = __builtin_amdgcn_readlane(c1, k) * tok;
        for (int64_t i = __builtin_amdgcn_readlane(c0, k) * tok + at; i < end; i += step)
          *(u32x4_t*)(a.out + i * 8) = u32x4_t{0u, 0u, 0u, 0u};
      }
    }
  }
}

// Tiles that T tokens of B sequences can make, and the state slots that their plan can use: with at most one
// item per compute unit one slot each, else two per half share of work, or the parts that long tiles may be cut into.
int64_t most_tiles(int64_t T, int64_t H, int64_t B, int nb) { return T * H / (32 * nb) + (B < T ? B : T); }
int64_t plan_slots(int64_t tiles, int cus, int64_t span) {
  if (tiles <= cus) return cus;
  const int64_t whole = 4 * (int64_t)cus + 64, most = kMostItems * (int64_t)cus, parts = kMostParts * tiles < most ? kMostParts * tiles : most;
  return span < 2 * kMinPart || parts < whole ? whole : parts;
}
// entries that a tile of these calls may visit
int64_t most_entries(int64_t rows, int64_t window, int64_t first, int64_t H) {
  const int64_t w = window + first + 128 + H;
  return window > 0 && w < rows ? w : rows;
}
// q rows per tile / 32: 64 where the sequences' q rows, on average, make no more tiles than 96 would, since such a tile has
// fewer products (and a wave free to convert fp8 rows); else 96, which read the rows less often.  Measured, 64 / 96: 64 q rows
// a sequence 157 / 161 us (32 sequences of 2 K to 32 K rows), up to 64 over fp8 110 / 157, 128 122 / 131 (fp8 104 / 133),
// 192 175 / 138, a 2048-token chunk 8.99 / 7.92 ms
int tile_blocks(int64_t T, int64_t H, int64_t B) {
  const int64_t r = (T * H + B - 1) / B;
  return (r + 63) / 64 <= (r + 95) / 96 ? 2 : 3;
}
bool plan_sizes(int64_t T, int64_t H, int64_t B) {
  return T >= 0 && H > 0 && B > 0 && T <= 0x7fffffff && H <= 0x7fffffff && B <= 0xfffff && T * H <= 0x7fffff80;
}

template <int D, int NB, bool FP8>
int launch_paged(const PagedArgs& a, int64_t tiles, hipStream_t st) {
  using G = GeoP<D, NB>;
  auto kern = paged_attn_kernel<D, NB, FP8>;
  static std::atomic<uint64_t> lds_attr{0};
  if (hipError_t e = smla_set_dynamic_lds((const void*)kern, G::LDS_BYTES, lds_attr); e != hipSuccess) return (int)e;
  const int64_t grid = tiles <= a.cus ? a.cus : tiles + a.slots;

  hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(64 * kWaves), G::LDS_BYTES, st, a);
  SMLA_HIP_CHECK_LAUNCH();
  const int64_t pieces = tiles * kUnits * NB * 2, most = 8 * (int64_t)a.cus;
  const dim3 grid2((unsigned)(pieces < most ? pieces : most));
  if (pieces >= 4 * (int64_t)a.cus)
    hipLaunchKernelGGL((paged_merge_kernel<D, NB, 4, 4>), grid2, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((paged_merge_kernel<D, NB, 1, kFewWaves>), grid2, dim3(64 * kFewWaves), 0, st, a);
  SMLA_HIP_CHECK_LAUNCH();
  return SMLA_OK;
}

}  // namespace
}  // namespace smla_attn

extern "C" size_t smla_paged_attn_workspace(int64_t T, int64_t H, int64_t B, int64_t rows, int64_t window,
                                            int64_t first) {
  using namespace smla_attn;
  if (!plan_sizes(T, H, B) || rows < 0 || window < 0 || first < 0) return 0;
  const int nb = tile_blocks(T, H, B);
  const int64_t state = nb == 2 ? GeoP<512, 2>::STATE_O + 4 * GeoP<512, 2>::STATE_F
                                : GeoP<512, 3>::STATE_O + 4 * GeoP<512, 3>::STATE_F;
  return (size_t)(kHeader + plan_slots(most_tiles(T, H, B, nb), smla_num_cus(), most_entries(rows, window, first, H)) * state);
}

extern "C" int smla_paged_attn_granted(const void* q, int q_dtype, const void* pages, int page_dtype,
                                       const float* page_scales, int64_t n_pages, int64_t P, const int32_t* table,
                                       int64_t ld_table, int64_t cols, const int32_t* lens, const int32_t* cu,
                                       const int32_t* granted, int64_t B, int64_t T, int64_t H, int64_t D, int64_t DV,
                                       float scale, const float* attn_sink, int64_t window, int64_t first, int flags,
                                       void* out, int out_dtype, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace smla_attn;
  if (!q || !pages || !table || !lens || !cu || !out) return SMLA_E_NULL;
  if (T < 0 || H <= 0 || B <= 0 || n_pages <= 0 || P <= 0 || cols <= 0 || ld_table < cols || D <= 0 || DV <= 0 || DV > D)
    return SMLA_E_SHAPE;
  if (q_dtype != SMLA_BF16 || out_dtype != SMLA_BF16 || (page_dtype != SMLA_BF16 && page_dtype != SMLA_FP8_E4M3))
    return SMLA_E_DTYPE;
  if (page_dtype == SMLA_FP8_E4M3 && !page_scales) return SMLA_E_NULL;
  if ((D != 512 && D != 576) || DV != 512) return SMLA_E_UNSUPPORTED;
  if (((uintptr_t)q | (uintptr_t)pages | (uintptr_t)out) & 15) return SMLA_E_UNSUPPORTED;
  if (window < 0 || first < 0 || window > 0x3fffffff || first > 0x3fffffff || (flags & ~SMLA_PAGED_FILL)) return SMLA_E_RANGE;
  if (!plan_sizes(T, H, B) || n_pages > 0x7fffffff || P > 0x7fffffff || n_pages * P > 0x7fffffff || cols > 0x7fffffff)
    return SMLA_E_RANGE;
  // rows of q are read while others of out are written
  const uintptr_t o0 = (uintptr_t)out, q0 = (uintptr_t)q;
  if (o0 < q0 + (uintptr_t)T * H * D * 2 && q0 < o0 + (uintptr_t)T * H * DV * 2) return SMLA_E_UNSUPPORTED;
  if (!usable_workspace(workspace, workspace_bytes, smla_paged_attn_workspace(T, H, B, cols * P, window, first))) return SMLA_E_WORKSPACE;
  if (T == 0) return SMLA_OK;
  PagedArgs a{};
  a.q = (const uint16_t*)q;
  a.pages = pages;
  a.page_scales = page_scales;
  a.table = table;
  a.lens = lens;
  a.cu = cu;
  a.granted = granted;
  a.sink = attn_sink;
  a.out = (uint16_t*)out;
  a.ws = (uint8_t*)workspace;
  a.ld_table = ld_table;
  a.T = (int)T;
  a.H = (int)H;
  a.B = (int)B;
  a.P = (int)P;
  a.n_pages = (int)n_pages;
  a.cols = (int)cols;
  a.window = (int)window;
  a.first = window > 0 ? (int)first : 0;
  a.cus = smla_num_cus();
  a.fill = (flags & SMLA_PAGED_FILL) != 0;
  a.scale = scale;
  const int nb = tile_blocks(T, H, B);
  const int64_t tiles = most_tiles(T, H, B, nb);
  a.slots = (int)plan_slots(tiles, a.cus, most_entries(cols * P, window, first, H));
  const hipStream_t st = (hipStream_t)stream;
  const bool fp8 = page_dtype == SMLA_FP8_E4M3;
#define SMLA_PAGED(DD, NB) return fp8 ? launch_paged<DD, NB, true>(a, tiles, st) : launch_paged<DD, NB, false>(a, tiles, st)
  if (nb == 2) {
    if (D == 576) SMLA_PAGED(576, 2);
    SMLA_PAGED(512, 2);
  }
  if (D == 576) SMLA_PAGED(576, 3);
  SMLA_PAGED(512, 3);
#undef SMLA_PAGED
}

extern "C" int smla_paged_attn(const void* q, int q_dtype, const void* pages, int page_dtype, const float* page_scales,
                               int64_t n_pages, int64_t P, const int32_t* table, int64_t ld_table, int64_t cols,
                               const int32_t* lens, const int32_t* cu, int64_t B, int64_t T, int64_t H, int64_t D,
                               int64_t DV, float scale, const float* attn_sink, int64_t window, int64_t first, int flags,
                               void* out, int out_dtype, void* workspace, size_t workspace_bytes, void* stream) {
  return smla_paged_attn_granted(q, q_dtype, pages, page_dtype, page_scales, n_pages, P, table, ld_table, cols, lens, cu,
                                 nullptr, B, T, H, D, DV, scale, attn_sink, window, first, flags, out, out_dtype,
                                 workspace, workspace_bytes, stream);
}
