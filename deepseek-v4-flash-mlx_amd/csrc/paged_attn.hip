// Attention of a ragged batch's newest tokens over a paged latent cache (absorbed MLA: every head reads the
// same rows).
//
// Token t of sequence b (cu[b] <= t < cu[b+1], n_b of them) sits at position p = lens[b] - n_b + (t - cu[b]) and
// attends the cache rows j <= p (row j: row j % P of page table[b, j / P]); with a window, those with
// j > p - window or j < first.  out = sum_j e^(s_j - m) row_j[:512] / (sum_j e^(s_j - m) + e^(sink - m)) with
// s_j = scale q.row_j; a token that sees no row gives 0.
//
// A sequence's (token, head) pairs are rows of q, n_b * H of them in a run; a tile is 64 of them (one token
// of 64 heads, four of 16).  The rows a tile visits are numbered through: entry e < nf is row e (the first
// rows, where the window starts behind them), entry e >= nf row lo + e - nf.  A work item is a run of `rps`
// entries of one tile; every workgroup finds its item from the lengths itself (no plan launch, no host
// read): with few tiles rps is the smallest that gives every compute unit at most one item, with many
// it only cuts entries that one workgroup would be long busy with.  Tiles of several items leave (m, l, O)
// states that paged_merge_kernel joins.
//
// The workgroup is the sparse decode kernel's: 12 waves, 4 that score 16 rows of q each (S^T = K Q^T,
// online softmax, P to LDS) and 8 that accumulate O^T += V^T P^T, one tile of 32 rows apart, rows copied
// HBM -> LDS into a ring by the value waves (fp8 rows: loaded, converted, written).  Row numbers come
// through an LDS ring of 8 tiles that score wave 0 fills seven tiles ahead, so a row list of any length
// costs one table read per row.
//
// Rows masked for some of a tile's q rows may hold anything (rows not yet written, pages of id -1 read as
// row 0): their probability is 0, and where a masked score is not finite the value waves take the tile's
// values with their infinities and NaN as 0 (a row that sees such a value has a NaN sum already).
#include "attn_common.h"

namespace smla_attn {
namespace {

typedef int32_t i32x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) i32x4_t lds_i32x4_t;
typedef __attribute__((address_space(3))) u32x2_t lds_u32x2_t;

constexpr int kTileQ = 64;       // q rows of a tile
constexpr int kIdTiles = 8;      // tiles of the row-number ring
constexpr int kMinRows = 64;     // fewest entries of an item
constexpr int kMinRowsMany = 256;  // the same with more tiles than compute units
constexpr int kHeader = 256;     // workspace bytes before the states

struct PagedArgs {
  const uint16_t* q;
  const void* pages;
  const float* page_scales;
  const int32_t *table, *lens, *cu;
  const float* sink;
  uint16_t* out;
  uint8_t* ws;
  int64_t ld_table;
  int T, H, B, P, n_pages, cols, window, first, cus, slots, fill;
  float scale;
};

template <int D, int NBUF_>
struct GeoP {
  static constexpr int ROWB = D * 2;
  static constexpr bool TAIL = D > 512;
  static constexpr int MSTRIDE = 1056;  // LDS bytes per row, columns 0..511
  static constexpr int MAIN_BYTES = kTileRows * MSTRIDE;
  static constexpr int TAIL_BYTES = TAIL ? kTileRows * 128 : 0;
  static constexpr int TILE_BYTES = MAIN_BYTES + TAIL_BYTES;
  static constexpr int NBUF = NBUF_;
  static constexpr int PSTRIDE = 80;  // bytes per q row in a P buffer: 32 probabilities, then padding (a flag in row 16 hg)
  static constexpr int PBUF = kTileQ * PSTRIDE;
  static constexpr int P_OFF = NBUF * TILE_BYTES;
  static constexpr int AL_OFF = P_OFF + 2 * PBUF;
  static constexpr int IDS_OFF = AL_OFF + 2 * kTileQ * 4;
  static constexpr int LOOP_END = IDS_OFF + kIdTiles * kTileRows * 4;
  static constexpr int STAGE = kTileQ * (1024 + 16);
  static constexpr int ML_OFF = LOOP_END > STAGE ? LOOP_END : STAGE;
  static constexpr int LDS_BYTES = ML_OFF + kTileQ * 2 * 4;
  static constexpr int NW = 12;
  static constexpr int KSTEPS = D / 32;
  static constexpr int NDMA = kTileRows + (TAIL ? kTileRows / 8 : 0);
  static_assert(LDS_BYTES <= 160 * 1024, "LDS budget");
  static_assert(NBUF >= 3, "Q takes the last two slots; tile 0 needs one more");
  static_assert(kIdTiles >= NBUF + 2, "row numbers are written before their copies are issued");
};

__device__ inline uint32_t pack2(float a, float b) { return pack_bf16x2(a, b); }

template <class Op>
__device__ inline float rows4_reduce(float v, Op op) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = op(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return op(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

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
  int tiles, span;  // tiles of 64 q rows; entries that a tile may visit
};

__device__ inline Seq load_seq(const PagedArgs& a, int b) {
  Seq s{0, 0, 0, 0, 0};
  if (b < a.B) {
    const int c0 = a.cu[b], c1 = a.cu[b + 1], len = a.lens[b];
    s.beg = min(max(c0, 0), a.T);
    s.n = max(min(c1, a.T) - s.beg, 0);
    s.len = max(len, 0);
    s.tiles = (int)(((uint32_t)s.n * (uint32_t)a.H + kTileQ - 1) / kTileQ);
    const int64_t cap = (int64_t)a.cols * a.P;
    int64_t span = s.len < cap ? s.len : cap;
    if (a.window > 0) {
      const int64_t w = (int64_t)a.window + a.first + (kTileQ + a.H - 1) / a.H;  // + 1 token - 1
      span = span < w ? span : w;
    }
    s.span = (int)span;
  }
  return s;
}

__device__ inline int ceil_div(int a, int b) { return (int)(((uint32_t)a + (uint32_t)b - 1) / (uint32_t)b); }
__device__ inline int splits_of(const Seq& s, int rps) { return max(1, ceil_div(s.span, rps)); }
__device__ inline int wave_sum_i(int v) { return __builtin_amdgcn_readlane(wave_incl_scan(v), 63); }

// Entries per item (a multiple of 32).  s0: sequences 0..63, kept in registers by the caller.
__device__ inline int plan_rps(const PagedArgs& a, const Seq& s0, int lane) {
  float work = 0.f;
  int tiles = 0, most = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const Seq s = b0 == 0 ? s0 : load_seq(a, b0 + lane);
    work += wave_sum_dpp((float)s.tiles * (float)s.span);
    tiles += wave_sum_i(s.tiles);
    most = max(most, (int)wave_max_dpp((float)(s.tiles > 0 ? s.span / kTileRows + 1 : 0)));
  }
  if (tiles > a.cus) {
    // more tiles than compute units: items of at most half a unit's share
    const float share = work / (float)(2 * a.cus * kTileRows);
    return max(kMinRowsMany, ((int)fminf(share, 16777216.f) + 1) * kTileRows);
  }
  // units of 32 entries: the fewest that give at most one item per compute unit
  int lo = max(kMinRows / kTileRows, (int)fminf(work / (float)(a.cus * kTileRows), 16777216.f));
  int hi = max(lo, most + (most >> 20) + 1);  // (most went through fp32)
  while (lo < hi) {
    const int mid = lo + (hi - lo) / 2;
    int items = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
      const Seq s = b0 == 0 ? s0 : load_seq(a, b0 + lane);
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
__device__ inline bool find_item(const PagedArgs& a, const Seq& s0, int lane, int rps, int w, bool by_tile, Item& it) {
  int before = 0, slots = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const Seq s = b0 == 0 ? s0 : load_seq(a, b0 + lane);
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

// states in the workspace: (m, l) of 64 rows per slot, then per slot a 64 KB block of O^T in bf16, in the
// order of the value waves' accumulators
__device__ inline float* state_ml(const PagedArgs& a, int slot) {
  return (float*)(a.ws + kHeader) + (int64_t)slot * (2 * kTileQ);
}
__device__ inline uint8_t* state_o(const PagedArgs& a, int slot) {
  return a.ws + kHeader + (int64_t)a.slots * (2 * kTileQ * 4) + (int64_t)slot * 65536;
}

constexpr int kDmaWaves = 8;
template <class G>
__device__ inline int dma_count(int w) {
  return w < 4 ? 0 : (G::NDMA - (w - 4) + kDmaWaves - 1) / kDmaWaves;
}

template <int D, int NBUF, bool FP8>
__global__ __launch_bounds__(768) void paged_attn_kernel(const PagedArgs a) {
  using G = GeoP<D, NBUF>;
  extern __shared__ __align__(16) uint8_t lds_generic[];
  lds_u8_t* lds = (lds_u8_t*)lds_generic;
  lds_i32_t* ids_s = (lds_i32_t*)(lds + G::IDS_OFF);
  lds_f32_t* al_s = (lds_f32_t*)(lds + G::AL_OFF);
  lds_f32_t* ml_s = (lds_f32_t*)(lds + G::ML_OFF);
  const uint32_t lds_base = (uint32_t)(uintptr_t)lds;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const bool scorer = wave < 4;
  const int g = lane >> 4, c = lane & 15;

  Item it;
  int rps;
  {
    const Seq s0 = load_seq(a, lane);
    rps = plan_rps(a, s0, lane);
    if (blockIdx.x == 0 && tid == 0) *(int*)a.ws = rps;
    if (!find_item(a, s0, lane, rps, blockIdx.x, false, it)) return;
  }
  if (it.nsplit > 1 && it.slot + it.nsplit > a.slots) return;  // lengths that no batch of T tokens has
  const int rows_b = it.s.n * a.H, m0 = it.tile * kTileQ;
  const int nh = min(kTileQ, rows_b - m0);  // q rows here
  const int64_t row0 = (int64_t)it.s.beg * a.H + m0;
  const int p0 = it.s.len - it.s.n;                                   // position of the first token
  const int p_lo = p0 + (int)((uint32_t)m0 / (uint32_t)a.H);           // of the tile's first and last
  const int p_hi = p0 + (int)((uint32_t)(m0 + nh - 1) / (uint32_t)a.H);
  const int w_lo = p_lo - a.window + 1;
  const int lo = a.window > 0 && w_lo > 0 ? w_lo : 0;
  const int nf = min(a.first, lo);
  const int64_t cap = (int64_t)a.cols * a.P;
  const int top = (int)min((int64_t)p_hi + 1, cap);  // rows below it
  const int entries = max(0, top - lo + nf);
  const int e_begin = it.split * rps, e_end = min(entries, e_begin + rps);
  const int ntiles = e_end > e_begin ? (e_end - e_begin + kTileRows - 1) / kTileRows : 0;
  const int32_t* trow = a.table + it.b * a.ld_table;
  // row number of entry e (-1: none, or a page id out of range)
  auto row_number = [&](int e) -> int {
    const int j = e < nf ? e : lo + (e - nf);
    int id = -1;
    if (e < e_end) {
      const uint32_t col = (uint32_t)j / (uint32_t)a.P;
      const int page = trow[col];
      if (page >= 0 && page < a.n_pages) id = page * a.P + (j - (int)col * a.P);
    }
    return id;
  };

  // ---- Q rows: two tiles of 32 in the last two ring slots (rows past nh read the tile's first)
  constexpr int QS = G::NBUF - 2;
  auto issue_rows = [&](int slot, auto&& rowp, bool nt) {
    const uint32_t tbase = lds_base + (uint32_t)(slot * G::TILE_BYTES);
    if (wave < 4) return;
#pragma unroll
    for (int k = 0; k < (G::NDMA + kDmaWaves - 1) / kDmaWaves; k++) {
      const int x = wave - 4 + kDmaWaves * k;
      if (x < kTileRows) {
        const uint32_t ld = __builtin_amdgcn_readfirstlane(tbase + x * G::MSTRIDE);
        if (nt)
          dma16_nt(rowp(x) + 16 * lane, ld);
        else
          dma16(rowp(x) + 16 * lane, ld);
      } else if (x < G::NDMA) {
        const int r0 = (x - kTileRows) * 8;
        const int r = r0 + (lane >> 3);
        const int ch = (lane & 7) ^ (r & 7);  // rope tails XOR-swizzled by row
        const uint32_t ld = __builtin_amdgcn_readfirstlane(tbase + G::MAIN_BYTES + r0 * 128);
        if (nt)
          dma16_nt(rowp(r) + 1024 + 16 * ch, ld);
        else
          dma16(rowp(r) + 1024 + 16 * ch, ld);
      }
    }
  };
  {
    const uint8_t* qrow0 = (const uint8_t*)(a.q + row0 * D);
    for (int qt = 0; qt < 2; qt++)
      issue_rows(
          QS + qt,
          [&](int r) {
            const int hl = 32 * qt + r;
            return qrow0 + (hl < nh ? hl : 0) * (int64_t)G::ROWB;
          },
          it.nsplit == 1);
  }
  // ---- the first eight tiles' row numbers, a score thread each
  if (scorer) ids_s[tid] = row_number(e_begin + tid);
  lds_barrier();

  auto issue_tile = [&](int tl) {
    if constexpr (!FP8) {
      const lds_i32_t* tid_s = ids_s + (tl % kIdTiles) * kTileRows;
      issue_rows(tl % G::NBUF,
                 [&](int r) { return (const uint8_t*)a.pages + (int64_t)max(tid_s[r], 0) * G::ROWB; }, false);
    }
  };
  const int my_dma = FP8 ? 0 : dma_count<G>(wave);

  // ---- fp8 rows: see attn_decode_kernel (16 codes per lane and chunk; main and rope columns apart)
  constexpr int F8_CH = D / 16;
  constexpr int F8_K = (kTileRows * F8_CH + 511) / 512;
  struct F8Regs {
    u32x4_t v[F8_K];
    float s[F8_K];
  };
  auto f8_chunk = [&](int vl, int k, int& r, int& cc) -> bool {
    if (k < 2) {
      const int ci = vl + 512 * k;
      r = ci >> 5;
      cc = ci & 31;
      return true;
    }
    r = vl >> 2;
    cc = 32 + (vl & 3);
    return vl < 128;
  };
  auto f8_load = [&](int tl, F8Regs& fr) {
    const lds_i32_t* tid_s = ids_s + (tl % kIdTiles) * kTileRows;
    const int vl = (wave - 4) * 64 + lane;
#pragma unroll
    for (int k = 0; k < F8_K; k++) {
      int r, cc;
      if (f8_chunk(vl, k, r, cc)) {
        const int64_t row = max(tid_s[r], 0);
        fr.v[k] = *(const u32x4_t*)((const uint8_t*)a.pages + row * D + 16 * cc);
        fr.s[k] = a.page_scales[row * (D / 64) + (cc >> 2)];
      }
    }
  };
  auto f8_store = [&](int tl, const F8Regs& fr) {
    lds_u8_t* slot = lds + (tl % G::NBUF) * G::TILE_BYTES;
    const int vl = (wave - 4) * 64 + lane;
#pragma unroll
    for (int k = 0; k < F8_K; k++) {
      int r, cc;
      if (f8_chunk(vl, k, r, cc)) {
        uint32_t w[8];
        // a normal power-of-two scale: code x scale is a bf16 value, given exactly by the scaled
        // converter; any other scale: the fp32 product rounded to bf16
        const uint32_t su = __float_as_uint(fr.s[k]);
        if ((su & 0x7fffffu) == 0 && su - 0x00800000u < 0x7f000000u) {
#pragma unroll
          for (int j = 0; j < 4; j++) {
            w[2 * j] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(fr.v[k][j], fr.s[k], false));
            w[2 * j + 1] =
                __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(fr.v[k][j], fr.s[k], true));
          }
        } else {
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const f32x2_t lo2 = __builtin_amdgcn_cvt_pk_f32_fp8((int)fr.v[k][j], false);
            const f32x2_t hi2 = __builtin_amdgcn_cvt_pk_f32_fp8((int)fr.v[k][j], true);
            w[2 * j] = pack_bf16x2(lo2.x * fr.s[k], lo2.y * fr.s[k]);
            w[2 * j + 1] = pack_bf16x2(hi2.x * fr.s[k], hi2.y * fr.s[k]);
          }
        }
        const u32x4_t w0 = {w[0], w[1], w[2], w[3]}, w1 = {w[4], w[5], w[6], w[7]};
        if (k < 2) {
          *(lds_u32x4_t*)(slot + r * G::MSTRIDE + 32 * cc) = w0;
          *(lds_u32x4_t*)(slot + r * G::MSTRIDE + 32 * cc + 16) = w1;
        } else {
          const int l0 = 2 * (cc - 32);
          *(lds_u32x4_t*)(slot + G::MAIN_BYTES + r * 128 + 16 * (l0 ^ (r & 7))) = w0;
          *(lds_u32x4_t*)(slot + G::MAIN_BYTES + r * 128 + 16 * ((l0 + 1) ^ (r & 7))) = w1;
        }
      }
    }
  };

  // ---- prologue copies: tiles 0 .. NBUF-3
  for (int tl = 0; tl < min(ntiles, QS); tl++) issue_tile(tl);
  F8Regs f8r;
  if constexpr (FP8) {
    if (!scorer) {
      for (int tl = 0; tl < min(ntiles, QS); tl++) {
        f8_load(tl, f8r);
        f8_store(tl, f8r);
      }
      if (QS < ntiles) f8_load(QS, f8r);
    }
  }
  wait_vm(FP8 ? 0 : max(0, min(QS, ntiles) - 1) * my_dma);
  lds_barrier();

  auto end_iteration = [&](int i) {
    if constexpr (!FP8) {
      if (i + 1 < ntiles) wait_vm(max(0, min(i + G::NBUF - 2, ntiles - 1) - (i + 1)) * my_dma);
    }
    lds_barrier();
    if (i + G::NBUF - 1 < ntiles) issue_tile(i + G::NBUF - 1);
  };

  if (scorer) {
    const int hg = wave;
    bf16x8_t qf[G::KSTEPS];
    {
      const lds_u8_t* qb = lds + (QS + (hg >> 1)) * G::TILE_BYTES;
      const int qr = (hg & 1) * 16 + c;
#pragma unroll
      for (int j = 0; j < G::KSTEPS; j++) {
        if (!G::TAIL || j < 16) {
          qf[j] = as_bf16x8(*(const lds_u32x4_t*)(qb + qr * G::MSTRIDE + 16 * g + 64 * j));
        } else {
          const int lch = 4 * (j - 16) + g;
          qf[j] = as_bf16x8(*(const lds_u32x4_t*)(qb + G::MAIN_BYTES + qr * 128 + 16 * (lch ^ (qr & 7))));
        }
      }
    }
    lds_barrier();  // Q slots free
    if (ntiles > QS) issue_tile(QS);
    // entries that q row 16 hg + c sees: e < eh, and e < first or e >= el
    const int m = min(m0 + hg * 16 + c, rows_b - 1);
    const int pc = p0 + (int)((uint32_t)m / (uint32_t)a.H);
    const int eh = pc + 1 - lo + nf;
    const int el = a.window > 0 ? pc - a.window + 1 - lo + nf : 0;
    // entries below eh_all and outside [first, el_all) are seen by every q row of the tile
    const int eh_all = p_lo + 1 - lo + nf, el_all = a.window > 0 ? p_hi - a.window + 1 - lo + nf : 0;
    float m_ref = -SMLA_INF, l_lane = 0.f;
    const int kq_off = c * G::MSTRIDE + 16 * g;
    // row numbers on their way: tile i + 7, read in iteration i - 1 and written in iteration i
    int next_id = 0;
    for (int i = 0; i <= ntiles; i++) {
      if (i < ntiles) {
        const lds_u8_t* buf = lds + (i % G::NBUF) * G::TILE_BYTES;
        auto ldk = [&](int j, int blk) -> u32x4_t {
          if (!G::TAIL || j < 16) return *(const lds_u32x4_t*)(buf + kq_off + blk * 16 * G::MSTRIDE + 64 * j);
          const int r = 16 * blk + c, lch = 4 * (j - 16) + g;
          return *(const lds_u32x4_t*)(buf + G::MAIN_BYTES + r * 128 + 16 * (lch ^ (r & 7)));
        };
        constexpr int PF = 6;
        u32x4_t ka[PF], kb[PF];
#pragma unroll
        for (int j = 0; j < PF; j++) {
          ka[j] = ldk(j, 0);
          kb[j] = ldk(j, 1);
        }
        __builtin_amdgcn_sched_barrier(0);
        if (wave == 0 && lane < kTileRows) {
          if (i > 0 && i + kIdTiles - 1 < ntiles) ids_s[((i + kIdTiles - 1) % kIdTiles) * kTileRows + lane] = next_id;
          if (i + kIdTiles < ntiles) next_id = row_number(e_begin + (i + kIdTiles) * kTileRows + lane);
        }
        f32x4_t s0 = {0.f, 0.f, 0.f, 0.f}, s1 = s0;
#pragma unroll
        for (int j = 0; j < G::KSTEPS; j++) {
          const u32x4_t a0 = ka[j % PF], a1 = kb[j % PF];
          if (j + PF < G::KSTEPS) {
            ka[j % PF] = ldk(j + PF, 0);
            kb[j % PF] = ldk(j + PF, 1);
          }
          s0 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(a0), qf[j], s0, 0, 0, 0);
          s1 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(a1), qf[j], s1, 0, 0, 0);
          __builtin_amdgcn_sched_barrier(0);
        }
        float x[8];
        const lds_i32_t* tid_s = ids_s + (i % kIdTiles) * kTileRows;
        const i32x4_t v0 = *(const lds_i32x4_t*)(tid_s + 4 * g);
        const i32x4_t v1 = *(const lds_i32x4_t*)(tid_s + 16 + 4 * g);
        const int e0 = e_begin + i * kTileRows;
        const bool open = e0 + kTileRows <= eh_all && (e0 >= el_all || e0 + kTileRows <= a.first);
        bool odd = false;  // a masked score that is not finite
        if (open) {
#pragma unroll
          for (int k = 0; k < 4; k++) {
            x[k] = v0[k] >= 0 ? s0[k] * a.scale : -SMLA_INF;
            x[4 + k] = v1[k] >= 0 ? s1[k] * a.scale : -SMLA_INF;
            odd |= (v0[k] < 0 && !(fabsf(s0[k]) < SMLA_INF)) | (v1[k] < 0 && !(fabsf(s1[k]) < SMLA_INF));
          }
        } else {
#pragma unroll
          for (int k = 0; k < 8; k++) {
            const int e = e0 + 4 * g + (k & 3) + 16 * (k >> 2);
            const int id = k < 4 ? v0[k & 3] : v1[k & 3];
            const float s = k < 4 ? s0[k & 3] : s1[k & 3];
            const bool ok = id >= 0 && e < eh && (e < a.first || e >= el);
            x[k] = ok ? s * a.scale : -SMLA_INF;
            odd |= !ok && !(fabsf(s) < SMLA_INF);
          }
        }
        const uint64_t any_odd = __builtin_amdgcn_ballot_w64(odd);
        float mt = x[0];
#pragma unroll
        for (int k = 1; k < 8; k++) mt = fmaxf(mt, x[k]);
        mt = rows4_reduce(mt, [](float x, float y) { return fmaxf(x, y); });
        float alpha = 1.f;
        if ((mt > m_ref + kRescaleSlack) || (m_ref == -SMLA_INF && mt > -SMLA_INF)) {
          alpha = (m_ref > -SMLA_INF) ? __expf(m_ref - mt) : 0.f;
          l_lane *= alpha;
          m_ref = mt;
        }
        float p[8];
#pragma unroll
        for (int k = 0; k < 8; k++) {
          // a NaN score stays NaN also where no maximum is set yet
          const float e = (m_ref > -SMLA_INF) ? __expf(x[k] - m_ref) : (x[k] == -SMLA_INF ? 0.f : x[k]);
          p[k] = bf16_round(e);
          l_lane += p[k];
        }
        lds_u8_t* pb = lds + G::P_OFF + (i & 1) * G::PBUF + (hg * 16 + c) * G::PSTRIDE;
        *(lds_u32x2_t*)(pb + 8 * g) = u32x2_t{pack2(p[0], p[1]), pack2(p[2], p[3])};
        *(lds_u32x2_t*)(pb + 32 + 8 * g) = u32x2_t{pack2(p[4], p[5]), pack2(p[6], p[7])};
        if (g == 0) al_s[(i & 1) * kTileQ + hg * 16 + c] = alpha;
        if (lane == 0) *(lds_i32_t*)(pb + 64) = any_odd != 0;
      }
      end_iteration(i);
    }
    const float l_tot = rows4_reduce(l_lane, [](float x, float y) { return x + y; });
    const int hl = hg * 16 + c;
    if (g == 0) {
      ml_s[hl * 2] = m_ref;
      ml_s[hl * 2 + 1] = l_tot;
      if (it.nsplit > 1) *(f32x2_t*)(state_ml(a, it.slot + it.split) + 2 * hl) = f32x2_t{m_ref, l_tot};
    }
    if (it.nsplit > 1) return;
    lds_barrier();  // (m, l) in LDS
    lds_barrier();  // the output block is staged
  } else {
    const int vw = wave - 4;
    const int hp = vw & 1, dq = vw >> 1;
    lds_barrier();  // pairs with the score waves' barrier after their Q^T reads
    if (ntiles > QS) issue_tile(QS);
    f32x16_t o[4];
#pragma unroll
    for (int mb = 0; mb < 4; mb++)
#pragma unroll
      for (int r = 0; r < 16; r++) o[mb][r] = 0.f;
    const int vj = lane >> 4, vJ = lane & 15;
    const int tr_off = (8 * (vj >> 1) + (vJ >> 2)) * G::MSTRIDE + 2 * (128 * dq + 16 * (vj & 1) + 4 * (vJ & 3));
    const int pr_off = (32 * hp + (lane & 31)) * G::PSTRIDE + 16 * (lane >> 5);
    for (int i = 0; i <= ntiles; i++) {
      if constexpr (FP8) {
        if (i + G::NBUF - 2 < ntiles) {
          f8_store(i + G::NBUF - 2, f8r);
          if (i + G::NBUF - 1 < ntiles) f8_load(i + G::NBUF - 1, f8r);
        }
      }
      if (i >= 1) {
        const int tp = i - 1;
        const lds_u8_t* buf = lds + (tp % G::NBUF) * G::TILE_BYTES;
        const lds_u8_t* pbuf = lds + G::P_OFF + (tp & 1) * G::PBUF;
        const float al = al_s[(tp & 1) * kTileQ + 32 * hp + (lane & 31)];
        const int odd = *(const lds_i32_t*)(pbuf + 32 * hp * G::PSTRIDE + 64) |
                        *(const lds_i32_t*)(pbuf + (32 * hp + 16) * G::PSTRIDE + 64);
        if (__builtin_amdgcn_ballot_w64(al != 1.f)) {
#pragma unroll
          for (int mb = 0; mb < 4; mb++) o[mb] *= al;
        }
        auto step = [&](bool clean) {
#pragma unroll
          for (int ks = 0; ks < 2; ks++) {
            const bf16x8_t pf = as_bf16x8(*(const lds_u32x4_t*)(pbuf + pr_off + 32 * ks));
            const lds_u8_t* vb = buf + tr_off + 16 * ks * G::MSTRIDE;
#pragma unroll
            for (int mb = 0; mb < 4; mb++) {
              const v4i16_t vlo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_t*)(vb + 64 * mb));
              const v4i16_t vhi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_t*)(vb + 64 * mb + 4 * G::MSTRIDE));
              bf16x8_t va = __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(vlo, vhi, 0, 1, 2, 3, 4, 5, 6, 7));
              if (clean) {
                u32x4_t w = __builtin_bit_cast(u32x4_t, va);
#pragma unroll
                for (int k = 0; k < 4; k++) w[k] = finite2(w[k]);
                va = as_bf16x8(w);
              }
              o[mb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(va, pf, o[mb], 0, 0, 0);
            }
          }
        };
        if (__builtin_amdgcn_readfirstlane(odd)) step(true);
        else step(false);
      }
      end_iteration(i);
    }
    if (it.nsplit > 1) {
      // O^T straight from the accumulators (attn_decode_kernel's order): 1 KB pieces ((vw * 4 + mb) * 2 + h),
      // in which lane l's 16 bytes are values 128 dq + 32 mb + 16 h + 8 (l >> 5) .. + 7 of q row 32 hp + (l & 31)
      uint8_t* blk = state_o(a, it.slot + it.split) + vw * 8192 + 16 * lane;
#pragma unroll
      for (int mb = 0; mb < 4; mb++) {
        uint32_t d[8];
#pragma unroll
        for (int k = 0; k < 8; k++) d[k] = pack2(o[mb][2 * k], o[mb][2 * k + 1]);
#pragma unroll
        for (int k = 0; k < 8; k += 4) {
          const auto x0 = __builtin_amdgcn_permlane32_swap(d[k], d[k + 2], false, false);
          const auto x1 = __builtin_amdgcn_permlane32_swap(d[k + 1], d[k + 3], false, false);
          const u32x4_t v4 = {x0[0], x1[0], x0[1], x1[1]};
          __builtin_nontemporal_store(v4, (u32x4_t*)(blk + (mb * 2 + (k >> 2)) * 1024));
        }
      }
      return;
    }
    lds_barrier();  // (m, l) in LDS
    const int hl = 32 * hp + (lane & 31);
    const float M = ml_s[hl * 2], L = ml_s[hl * 2 + 1];
    float inv = 0.f;  // no row seen: 0
    if (!(L == 0.f)) {
      const float snk = a.sink && hl < nh ? a.sink[(uint32_t)(m0 + hl) % (uint32_t)a.H] : -SMLA_INF;
      inv = 1.0f / (L + (snk == -SMLA_INF ? 0.f : __expf(snk - M)));
    }
    const int dvb = 128 * dq + 4 * (lane >> 5);
    lds_u8_t* srow = lds + hl * (1024 + 16);
#pragma unroll
    for (int mb = 0; mb < 4; mb++)
#pragma unroll
      for (int qd = 0; qd < 4; qd++) {
        const f32x4_t v = f32x4_t{o[mb][4 * qd], o[mb][4 * qd + 1], o[mb][4 * qd + 2], o[mb][4 * qd + 3]} * inv;
        *(lds_u32x2_t*)(srow + 2 * (dvb + 32 * mb + 8 * qd)) = u32x2_t{pack2(v[0], v[1]), pack2(v[2], v[3])};
      }
    lds_barrier();
  }
  // the tile's q rows are consecutive rows of out
  uint8_t* dst = (uint8_t*)(a.out + row0 * 512);
  for (int i = tid; i < nh * 64; i += G::NW * 64)
    __builtin_nontemporal_store(*(const lds_u32x4_t*)(lds + (i >> 6) * (1024 + 16) + (i & 63) * 16),
                                (u32x4_t*)(dst + (int64_t)i * 16));
}

// ---------------------------------------------------------------------------------------------
// Joins the states of split tiles: a workgroup of 4 waves takes a 1 KB piece (8 values of 64 q rows' half)
// of one tile, wave w the splits w, w + 4, .. eight at a time with a running maximum, the waves' sums then
// through LDS in a fixed order.  Workgroups walk the pieces of all split tiles; with `fill` they also clear
// the rows behind the last sequence.
constexpr int kMergeWaves = 4, kMergeBatch = 8;

__global__ __launch_bounds__(64 * kMergeWaves) void paged_merge_kernel(const PagedArgs a) {
  __shared__ float red[kMergeWaves][64][10];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const Seq s0 = load_seq(a, lane);
  const int rps = __builtin_amdgcn_readfirstlane(*(const int*)a.ws);
  for (int64_t w = blockIdx.x;; w += gridDim.x) {
    Item it;
    if (!find_item(a, s0, lane, rps, (int)(w >> 6), true, it)) break;
    if (it.slot + it.nsplit > a.slots) continue;
    const int piece = (int)(w & 63);
    const int row = 32 * ((piece >> 3) & 1) + (lane & 31);  // vw = piece / 8: hp = vw & 1, dq = vw >> 1
    float m = -SMLA_INF, l = 0.f, acc[8];
#pragma unroll
    for (int k = 0; k < 8; k++) acc[k] = 0.f;
    for (int sp0 = wave; sp0 < it.nsplit; sp0 += kMergeWaves * kMergeBatch) {
      f32x2_t ml[kMergeBatch];
      u32x4_t v[kMergeBatch];
#pragma unroll
      for (int k = 0; k < kMergeBatch; k++) {
        const int sp = sp0 + kMergeWaves * k;
        if (sp < it.nsplit) {
          ml[k] = *(const f32x2_t*)(state_ml(a, it.slot + sp) + 2 * row);
          v[k] = *(const u32x4_t*)(state_o(a, it.slot + sp) + piece * 1024 + 16 * lane);
        }
      }
      float top = m;
#pragma unroll
      for (int k = 0; k < kMergeBatch; k++)
        if (sp0 + kMergeWaves * k < it.nsplit) top = fmaxf(top, ml[k][0]);
      const float keep = m > -SMLA_INF ? __expf(m - top) : (top == m ? 1.f : 0.f);
      l *= keep;
#pragma unroll
      for (int j = 0; j < 8; j++) acc[j] *= keep;
      m = top;
#pragma unroll
      for (int k = 0; k < kMergeBatch; k++)
        if (sp0 + kMergeWaves * k < it.nsplit) {
          // a state without a maximum has l = 0 (nothing seen) or NaN
          const float e = ml[k][0] > -SMLA_INF ? __expf(ml[k][0] - m) : 1.f;
          l += ml[k][1] * e;
#pragma unroll
          for (int j = 0; j < 4; j++) {
            acc[2 * j] += __uint_as_float(v[k][j] << 16) * e;
            acc[2 * j + 1] += __uint_as_float(v[k][j] & 0xffff0000u) * e;
          }
        }
    }
    __syncthreads();  // the last piece's sums are read
    red[wave][lane][0] = m;
    red[wave][lane][1] = l;
#pragma unroll
    for (int j = 0; j < 8; j++) red[wave][lane][2 + j] = acc[j];
    __syncthreads();
    if (wave == 0) {
      float top = m;
#pragma unroll
      for (int k = 1; k < kMergeWaves; k++) top = fmaxf(top, red[k][lane][0]);
      float sum = 0.f, y[8];
#pragma unroll
      for (int j = 0; j < 8; j++) y[j] = 0.f;
#pragma unroll
      for (int k = 0; k < kMergeWaves; k++) {
        const float mk = red[k][lane][0], e = mk > -SMLA_INF ? __expf(mk - top) : 1.f;
        sum += red[k][lane][1] * e;
#pragma unroll
        for (int j = 0; j < 8; j++) y[j] += red[k][lane][2 + j] * e;
      }
      const int m0 = it.tile * kTileQ, rows_b = it.s.n * a.H;
      if (m0 + row < rows_b) {
        float inv = 0.f;
        if (!(sum == 0.f)) {
          const float snk = a.sink ? a.sink[(uint32_t)(m0 + row) % (uint32_t)a.H] : -SMLA_INF;
          inv = 1.0f / (sum + (snk == -SMLA_INF ? 0.f : __expf(snk - top)));
        }
        const int vw = piece >> 3, dv = 128 * (vw >> 1) + 32 * ((piece >> 1) & 3) + 16 * (piece & 1) + 8 * (lane >> 5);
        u32x4_t o;
#pragma unroll
        for (int j = 0; j < 4; j++) o[j] = pack2(y[2 * j] * inv, y[2 * j + 1] * inv);
        *(u32x4_t*)(a.out + ((int64_t)it.s.beg * a.H + m0 + row) * 512 + dv) = o;
      }
    }
  }
  if (a.fill) {
    const int64_t from = (int64_t)min(max(a.cu[a.B], 0), a.T) * a.H * 64, to = (int64_t)a.T * a.H * 64;
    for (int64_t i = from + (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < to; i += (int64_t)gridDim.x * blockDim.x)
      *(u32x4_t*)(a.out + i * 8) = u32x4_t{0u, 0u, 0u, 0u};
  }
}

template <int D, int NBUF, bool FP8>
int launch_paged(const PagedArgs& a, int64_t grid, hipStream_t st) {
  using G = GeoP<D, NBUF>;
  auto kern = paged_attn_kernel<D, NBUF, FP8>;
  static std::atomic<uint64_t> lds_attr{0};
  if (hipError_t e = smla_set_dynamic_lds((const void*)kern, G::LDS_BYTES, lds_attr); e != hipSuccess) return (int)e;
  hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(G::NW * 64), G::LDS_BYTES, st, a);
  SMLA_HIP_CHECK_LAUNCH();
  return SMLA_OK;
}

// Tiles that T tokens of B sequences can make, and the state slots that their plan can use: with at most one
// item per compute unit one slot each, else two per half share of work.
int64_t most_tiles(int64_t T, int64_t H, int64_t B) { return T * H / kTileQ + (B < T ? B : T); }
int64_t plan_slots(int64_t T, int64_t H, int64_t B, int cus) {
  return most_tiles(T, H, B) <= cus ? cus : 4 * (int64_t)cus + 64;
}
bool plan_sizes(int64_t T, int64_t H, int64_t B) {
  return T >= 0 && H > 0 && B > 0 && T <= 0x7fffffff && H <= 0x7fffffff && B <= 0xfffff && T * H <= 0x7fffffc0;
}

}  // namespace
}  // namespace smla_attn

extern "C" size_t smla_paged_attn_workspace(int64_t T, int64_t H, int64_t B) {
  using namespace smla_attn;
  if (!plan_sizes(T, H, B)) return 0;
  return (size_t)(kHeader + plan_slots(T, H, B, smla_num_cus()) * (2 * kTileQ * 4 + 65536));
}

extern "C" int smla_paged_attn(const void* q, int q_dtype, const void* pages, int page_dtype, const float* page_scales,
                               int64_t n_pages, int64_t P, const int32_t* table, int64_t ld_table, int64_t cols,
                               const int32_t* lens, const int32_t* cu, int64_t B, int64_t T, int64_t H, int64_t D,
                               int64_t DV, float scale, const float* attn_sink, int64_t window, int64_t first, int flags,
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
  if (!usable_workspace(workspace, workspace_bytes, smla_paged_attn_workspace(T, H, B))) return SMLA_E_WORKSPACE;
  if (T == 0) return SMLA_OK;
  PagedArgs a{};
  a.q = (const uint16_t*)q;
  a.pages = pages;
  a.page_scales = page_scales;
  a.table = table;
  a.lens = lens;
  a.cu = cu;
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
  a.slots = (int)plan_slots(T, H, B, a.cus);
  a.fill = (flags & SMLA_PAGED_FILL) != 0;
  a.scale = scale;
  const int64_t tiles = most_tiles(T, H, B);
  const int64_t grid = tiles <= a.cus ? a.cus : tiles + 2 * (int64_t)a.cus + 64;
  const hipStream_t st = (hipStream_t)stream;
  int rc;
  if (page_dtype == SMLA_FP8_E4M3)
    rc = D == 576 ? launch_paged<576, 3, true>(a, grid, st) : launch_paged<512, 3, true>(a, grid, st);
  else
    rc = D == 576 ? launch_paged<576, 3, false>(a, grid, st) : launch_paged<512, 3, false>(a, grid, st);
  if (rc != 0) return rc;
  const int64_t pieces = tiles * 64, most = 8 * (int64_t)a.cus;
  hipLaunchKernelGGL(paged_merge_kernel, dim3((unsigned)(pieces < most ? pieces : most)), dim3(64 * kMergeWaves), 0, st, a);
  SMLA_HIP_CHECK_LAUNCH();
  return SMLA_OK;
}
