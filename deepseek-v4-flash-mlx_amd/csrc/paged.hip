// The paged latent cache beside its attention: rows written into pages, slots forked and grown, pages
// moved together.
//
// A pool holds n_pages pages of P rows of D channels; sequence (slot) b keeps its rows in the pages
// table[b, 0 ..], row j in row j % P of page table[b, j / P].  Pages may be shared between slots (refs
// counts the table entries and other holders of a page; 0: free).
//
//  * paged_append_kernel : per new token, the per-head RMS norm and RoPE of its query heads and the norm,
//                          RoPE and quantisation of its latent row, written to the row's page.  One wave
//                          per (token, head) row; nothing is read twice.
//  * update_one / update_plan + update_apply : slot s becomes a copy of slot parent[s] plus (or less) grow[s] rows.
//  * compact_one / compact_plan + compact_apply : live pages moved to the pool's first ids.
#include "smla_internal.h"

namespace {

// ---------------------------------------------------------------------------------------------
// append
struct AppendArgs {
  const void* q;   // [T, H, D], tokens ldq elements apart
  const void* kv;  // [T, D], tokens ldkv elements apart
  int64_t ldq, ldkv;
  uint32_t T, H, rows_per_tok;  // rows_per_tok = H + 1 (the latent row last)
  int D, norm_dims, rd, flags, sim, page_dtype;
  const float *q_w, *kv_w, *cos_t, *sin_t;
  int64_t n_pos;
  float eps;
  uint16_t* q_out;
  void* pages;
  float* scales;
  int n_pages, P, cols, B;
  int64_t ld_table;
  const int32_t *table, *lens, *cu, *granted;  // granted null: every sequence
};

// Sequence of token t (the number of sequences that end at or before it; B: behind the last) and its
// position, by one wave: every lane reads one boundary and one length, in one round trip per 64
// sequences.  false: a token of no sequence, or of one that was not granted its rows.
__device__ inline bool token_position(const AppendArgs& a, int t, int lane, int& seq, int64_t& pos) {
  seq = 0;
  int beg = 0, end = 0, len = 0, has = 1;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const int b = b0 + lane;
    int c0 = 0, c1 = 0x7fffffff, n = 0, g = 1;
    if (b < a.B) {
      c0 = a.cu[b];
      c1 = a.cu[b + 1];
      n = a.lens[b];
      if (a.granted) g = a.granted[b];
    }
    const uint64_t done = __builtin_amdgcn_ballot_w64(c1 <= t);
    const int k = (int)__builtin_popcountll(done);
    seq += k;
    if (k < 64) {
      beg = __builtin_amdgcn_readlane(c0, k);
      end = __builtin_amdgcn_readlane(c1, k);
      len = __builtin_amdgcn_readlane(n, k);
      has = __builtin_amdgcn_readlane(g, k);
      break;
    }
  }
  if (seq >= a.B || beg > t || beg < 0 || has == 0) return false;
  pos = (int64_t)len - ((int64_t)end - beg) + (t - beg);
  return pos >= 0;
}

template <int XDT>
__device__ inline f32x4_t load4(const void* p, int64_t i) {
  if constexpr (XDT == SMLA_F32) {
    return *(const f32x4_t*)((const float*)p + i);
  } else {
    const u32x2_t w = *(const u32x2_t*)((const uint16_t*)p + i);
    return f32x4_t{__uint_as_float(w[0] << 16), __uint_as_float(w[0] & 0xffff0000u), __uint_as_float(w[1] << 16),
                   __uint_as_float(w[1] & 0xffff0000u)};
  }
}

// Lane l of a wave owns channels 256 c + 4 l .. + 3 of chunk c: every access of a wave is one contiguous
// run, a rotation pair and a lane's norm weights stay in the lane, and a 64-channel quantisation block
// is one 16-lane row.  Sums and the rotation are fp32; a result is rounded once, to its stored type.
// Bound by HBM: 4096 tokens of 64 heads and a row (fp32 in, bf16 out, 818 MB) 142 us = 5.8 TB/s; 8 tokens 3.6 us, latency.
template <int XDT, int NCH>
__global__ __launch_bounds__(256) void paged_append_kernel(const AppendArgs a) {
  const int lane = threadIdx.x & 63;
  const uint32_t r = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
  const uint32_t t = r / a.rows_per_tok;
  if (t >= a.T) return;
  const uint32_t h = r - t * a.rows_per_tok;
  const bool is_q = h < a.H;
  const int D = a.D;
  f32x4_t v[NCH];
  {
    const void* src = is_q ? a.q : a.kv;
    const int64_t at = is_q ? (int64_t)t * a.ldq + (int64_t)h * D : (int64_t)t * a.ldkv;
#pragma unroll
    for (int c = 0; c < NCH; c++) {
      const int ch = 256 * c + 4 * lane;
      v[c] = ch < D ? load4<XDT>(src, at + ch) : f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
  }
  int seq;
  int64_t pos = 0;
  bool live = token_position(a, (int)t, lane, seq, pos);
  if (live && a.rd > 0 && pos >= a.n_pos) live = false;
  uint16_t* qo = a.q_out + ((int64_t)t * a.H + h) * D;
  if (!live) {
    if (is_q && (a.flags & SMLA_PAGED_FILL)) {
#pragma unroll
      for (int c = 0; c < NCH; c++) {
        const int ch = 256 * c + 4 * lane;
        if (ch < D) *(u32x2_t*)(qo + ch) = u32x2_t{0u, 0u};
      }
    }
    return;
  }
  const int nope = D - a.rd;
  // the row's page (latent rows), the rotation of the rope channels: read before the norm's reduction
  int page = -1;
  if (!is_q) {
    const int64_t col = (int64_t)((uint32_t)pos / (uint32_t)a.P);
    if (col < a.cols) page = a.table[seq * a.ld_table + col];
  }
  f32x2_t cs[NCH], sn[NCH];
  f32x4_t w[NCH];
  const bool norm = (a.flags & (is_q ? SMLA_PAGED_NORM_Q : SMLA_PAGED_NORM_KV)) != 0;
  const float* nw = is_q ? a.q_w : a.kv_w;
#pragma unroll
  for (int c = 0; c < NCH; c++) {
    const int ch = 256 * c + 4 * lane;
    cs[c] = f32x2_t{1.f, 1.f};
    sn[c] = f32x2_t{0.f, 0.f};
    if (ch >= nope && ch < D) {
      const int64_t i = pos * (a.rd / 2) + ((ch - nope) >> 1);
      cs[c] = f32x2_t{a.cos_t[i], a.cos_t[i + 1]};
      sn[c] = f32x2_t{a.sin_t[i], a.sin_t[i + 1]};
    }
    w[c] = f32x4_t{1.f, 1.f, 1.f, 1.f};
    if (norm && nw && ch < a.norm_dims) w[c] = f32x4_t{nw[ch], nw[ch + 1], nw[ch + 2], nw[ch + 3]};
  }
  if (norm) {
    float ss = 0.f;
#pragma unroll
    for (int c = 0; c < NCH; c++)
      if (256 * c + 4 * lane < a.norm_dims)
        ss += (v[c][0] * v[c][0] + v[c][1] * v[c][1]) + (v[c][2] * v[c][2] + v[c][3] * v[c][3]);
    const float inv = rsqrtf(wave_sum_dpp(ss) / (float)a.norm_dims + a.eps);
#pragma unroll
    for (int c = 0; c < NCH; c++)
      if (256 * c + 4 * lane < a.norm_dims)
#pragma unroll
        for (int k = 0; k < 4; k++) v[c][k] = w[c][k] * (v[c][k] * inv);
  }
#pragma unroll
  for (int c = 0; c < NCH; c++) {
    if (256 * c + 4 * lane >= nope) {
      const f32x4_t x = v[c];
      v[c] = f32x4_t{x[0] * cs[c][0] - x[1] * sn[c][0], x[0] * sn[c][0] + x[1] * cs[c][0],
                     x[2] * cs[c][1] - x[3] * sn[c][1], x[2] * sn[c][1] + x[3] * cs[c][1]};
    }
  }
  if (is_q) {
#pragma unroll
    for (int c = 0; c < NCH; c++) {
      const int ch = 256 * c + 4 * lane;
      if (ch < D) *(u32x2_t*)(qo + ch) = u32x2_t{pack_bf16x2(v[c][0], v[c][1]), pack_bf16x2(v[c][2], v[c][3])};
    }
    return;
  }
  const int64_t row = (int64_t)page * a.P + (uint32_t)pos % (uint32_t)a.P;
  const bool stored = page >= 0 && page < a.n_pages;
#pragma unroll
  for (int c = 0; c < NCH; c++) {
    const int ch = 256 * c + 4 * lane;
    // per 64 channels: s = 2^ceil(log2(max(|y|, 1e-4) / 448)), code = e4m3(y / s) to nearest even (NaN, as the whole block's
    // value, where the largest is not finite: the page shows what a bf16 page would)
    const bool coded = a.page_dtype == SMLA_FP8_E4M3 || (a.sim == SMLA_SIM_FP8 && ch < nope);
    f32x4_t y = v[c];
    uint32_t m = max(max(mag_bits(y[0]), mag_bits(y[1])), max(mag_bits(y[2]), mag_bits(y[3])));
    m = max(m, dpp_u<0xB1>(m));
    m = max(m, dpp_u<0x4E>(m));
    m = max(m, dpp_u<0x141>(m));
    m = max(m, dpp_u<0x140>(m));
    const float s = fp8_scale(m);
    if (ch >= D || !stored) continue;
    if (coded) {
      float z[4];
#pragma unroll
      for (int k = 0; k < 4; k++) z[k] = fminf(fmaxf(y[k] / s, -448.f), 448.f);
      int code = __builtin_amdgcn_cvt_pk_fp8_f32(z[0], z[1], 0, false);
      code = __builtin_amdgcn_cvt_pk_fp8_f32(z[2], z[3], code, true);
      if (m >= kNotFinite) code = kNanCodes;
      if (a.page_dtype == SMLA_FP8_E4M3) {
        *(int*)((uint8_t*)a.pages + row * D + ch) = code;
        if ((lane & 15) == 0) a.scales[row * (D / 64) + ch / 64] = s;
        continue;
      }
      const f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8(code, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(code, true);
      y = f32x4_t{lo[0] * s, lo[1] * s, hi[0] * s, hi[1] * s};
    }
    *(u32x2_t*)((uint16_t*)a.pages + row * D + ch) = u32x2_t{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
  }
}

// ---------------------------------------------------------------------------------------------
// pages: shared pieces
constexpr int kPlanThreads = 1024;
constexpr int kWavePages = 1024;        // most pages of a wave in one step of a scan over refs
constexpr int kStepPages = kPlanThreads / 64 * kWavePages;
constexpr int64_t kCopyChunk = 8192;    // bytes of one copy item (16384 leave larger remainders of pages: 61.8 us below for 55.4)
constexpr int kCopyThreads = 256;       // threads that copy an item together
// One launch does all where every workgroup can plan for itself: inputs are read only, so that all plans agree, and the plan
// fits the LDS: pools of one scan step, up to 1024 slots, and few enough table entries for one workgroup.  Measured
// against two launches: 32 slots of 128 entries and 1500 pages 7.2 us (4.6 + 3.3), 300 pages moved together 7.3 us (7.1 + 4.0),
// 8192 pages 69.7 us (16.5 + 60.3), and a launch less for the host, 3 us; since then the copies' chunks and nontemporal accesses
// took the last to 55 us.  Larger ones are planned once.
constexpr int64_t kOneEntries = 32768;

// Exclusive prefix sum of v over the workgroup (16 waves); total: the sum.
__device__ inline int block_excl(int v, int* red, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int incl = wave_incl_scan(v);
  __syncthreads();
  if (lane == 63) red[wave] = incl;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 64; w++) {
    const int x = red[w];
    before += w < wave ? x : 0;
    total += x;
  }
  return before + incl - v;
}

__device__ inline int wave_id() { return __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6); }

// A wave's share of a scan over refs: `per` pages (a multiple of 64) from base on, a coalesced load and a ballot per 64; bit l of
// m[k] for page base + 64 k + l: a free page (refs 0) or a live one (refs > 0).  v: the counts, 0 past the pages n.
constexpr int kBallots = kWavePages / 64;
template <bool FREE>
__device__ inline int wave_pages(const int32_t* refs, int64_t n, int64_t base, int per, int (&v)[kBallots],
                                 uint64_t (&m)[kBallots]) {
  const int lane = threadIdx.x & 63, left = (int)min(max(n - base, (int64_t)0), (int64_t)per);
  const int32_t* at = refs + min(base, n - 1);
  int sum = 0;
#pragma unroll
  for (int k = 0; k < kBallots; k++) v[k] = 64 * k + lane < left ? at[64 * k + lane] : 0;
#pragma unroll
  for (int k = 0; k < kBallots; k++) {
    m[k] = __builtin_amdgcn_ballot_w64(FREE ? (v[k] == 0) & (64 * k + lane < left) : v[k] > 0);
    sum += (int)__builtin_popcountll(m[k]);
  }
  return sum;
}
// pages of a wave where 16 share n of them (one step)
__device__ inline int per_wave(int n) { return (n + kPlanThreads - 1) / kPlanThreads * 64; }
// Sums of a wave-uniform x over the waves before this one (returned) and over all (total).
__device__ inline int waves_excl(int x, int* red, int& total) {
  const int wave = wave_id();
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[wave] = x;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 64; w++) {
    before += w < wave ? red[w] : 0;
    total += red[w];
  }
  return before;
}
// set bits of m below bit k (0 and less: none, 64 and more: all)
__device__ inline int bits_below(uint64_t m, int64_t k) {
  return k <= 0 ? 0 : (int)__builtin_popcountll(k >= 64 ? m : m & ((1ull << k) - 1));
}
__device__ inline int lane_below(uint64_t m) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
}

struct Pool {
  uint8_t* base;
  int64_t layer_bytes;
  int64_t page_bytes, row_bytes;
};

// n bytes by kCopyThreads threads, 16 at a time where both sides are aligned.  NT: not kept in the caches (whole pages of a
// pool that is larger than those: 8192 pages of 64 x 576 61.8 us against 69.0; a fork's tail page is read soon and stays).
template <bool NT>
__device__ inline void copy_span(uint8_t* dst, const uint8_t* src, int64_t n) {
  const int tid = threadIdx.x % kCopyThreads;
  const uintptr_t mix = (uintptr_t)dst | (uintptr_t)src;
  if ((mix & 15) == 0) {
    constexpr int kLoads = (int)(kCopyChunk / (16 * kCopyThreads));
    const int64_t nv = n / 16;
    const u32x4_t* from = (const u32x4_t*)src;
    u32x4_t* to = (u32x4_t*)dst;
    for (int64_t i = tid; i < nv; i += kLoads * kCopyThreads) {
      u32x4_t v[kLoads];
#pragma unroll
      for (int k = 0; k < kLoads; k++)
        if (i + k * kCopyThreads < nv) {
          if constexpr (NT) v[k] = __builtin_nontemporal_load(from + i + k * kCopyThreads);
          else v[k] = from[i + k * kCopyThreads];
        }
#pragma unroll
      for (int k = 0; k < kLoads; k++)
        if (i + k * kCopyThreads < nv) {
          if constexpr (NT) __builtin_nontemporal_store(v[k], to + i + k * kCopyThreads);
          else to[i + k * kCopyThreads] = v[k];
        }
    }
    for (int64_t i = nv * 16 + tid; i < n; i += kCopyThreads) dst[i] = src[i];
  } else if (((mix | (uintptr_t)n) & 3) == 0) {
    for (int64_t i = tid; i < n / 4; i += kCopyThreads) ((uint32_t*)dst)[i] = ((const uint32_t*)src)[i];
  } else {
    for (int64_t i = tid; i < n; i += kCopyThreads) dst[i] = src[i];
  }
}

// chunk `part` of the first `rows` rows of page src copied to page dst, in layer `layer`: the parts
// below `parts` cover the first pool in kCopyChunk pieces, part `parts` the second pool (if any)
template <bool NT>
__device__ inline void copy_item(const Pool& p0, const Pool& p1, int layer, int64_t src, int64_t dst, int64_t rows,
                                 int64_t part, int64_t parts) {
  if (part < parts) {
    const int64_t all = rows * p0.row_bytes, from = part * kCopyChunk;
    if (from >= all) return;
    uint8_t* b = p0.base + layer * p0.layer_bytes + from;
    copy_span<NT>(b + dst * p0.page_bytes, b + src * p0.page_bytes, all - from < kCopyChunk ? all - from : kCopyChunk);
  } else {
    uint8_t* b = p1.base + layer * p1.layer_bytes;
    copy_span<NT>(b + dst * p1.page_bytes, b + src * p1.page_bytes, rows * p1.row_bytes);
  }
}

struct PageArgs {
  const int32_t *table, *lens, *refs, *parent, *grow;
  int64_t ld_table;
  int S, M, n_pages, P, layers;
  int32_t *table_out, *lens_out, *refs_out, *granted, *live;
  Pool p0, p1;  // p1.base null: none
  int64_t parts, items_per_copy;
  int32_t* ws;
};

// What slot s asks for: rows taken from its parent (all, or those that a negative grow leaves), rows afterwards, entries
// taken from the parent as they are, pages afterwards; false: an argument out of range.
struct SlotNeed {
  int rows, next, full, pages, parent;
};
__device__ inline bool slot_need(const PageArgs& a, int s, SlotNeed& n) {
  const int p = a.parent[s], g = a.grow[s];
  if (p < -1 || p >= a.S) return false;
  const int have = p >= 0 ? a.lens[p] : 0;
  n.parent = p;
  const int64_t next = (int64_t)have + g;
  if (have < 0 || next < 0 || next > 0x7fffffff) return false;
  n.next = (int)next;
  n.rows = min(have, n.next);
  const uint32_t P = (uint32_t)a.P;
  const int64_t pages = (next + P - 1) / P;
  n.pages = (int)pages;
  const uint32_t whole = (uint32_t)n.rows / P;
  n.full = (int)whole;
  if (pages > a.M) return false;
  if (p == s && (uint32_t)n.rows % P) {
    // its own partly filled page stays, unless rows change in one that others hold too (a slot that gave rows back past a
    // fork): that is copied like another slot's
    const int page = g != 0 ? a.table[s * a.ld_table + whole] : -1;
    if (page < 0 || page >= a.n_pages || a.refs[page] <= 1) n.full++;
  }
  return true;
}
__device__ inline int tail_rows(const PageArgs& a, const SlotNeed& n) {
  return (int)max((int64_t)n.rows - (int64_t)n.full * a.P, (int64_t)0);
}

// What becomes of slot s: its first fresh rank (-1: refused), the slot it copies, entries it shares with that, entries
// afterwards and before, rows of a tail page to copy (0: none).
struct SlotPlan {
  int at, parent, full, pages, held, tail;
};
__device__ inline SlotPlan slot_plan(const PageArgs& a, int s, int at, const SlotNeed& n) {
  const int len = a.lens[s];
  return SlotPlan{at, n.parent, n.full, n.pages, len > 0 ? (int)(((uint32_t)len + (uint32_t)a.P - 1) / (uint32_t)a.P) : 0,
                  tail_rows(a, n)};
}
// Entry c of slot s after the update, fresh(k) the fresh page of rank k; count(page, by) for every change of a page's holders.
template <class Fresh, class Count>
__device__ inline int slot_entry(const PageArgs& a, int s, int c, const SlotPlan& n, Fresh&& fresh, Count&& count) {
  const int old = a.table[s * a.ld_table + c];
  if (n.at < 0) return old;
  const int now = c < n.full ? a.table[n.parent * a.ld_table + c] : c < n.pages ? fresh(n.at + c - n.full) : -1;
  if (n.parent != s || c >= n.full) {  // (a kept slot's first entries stay as they are)
    if (c < n.held) count(old, -1);
    if (c < n.pages) count(now, 1);
  }
  return now;
}
// the tail page of a slot: item `part` of layer `layer` of its copy to page dst
__device__ inline void copy_tail(const PageArgs& a, const SlotPlan& n, int64_t dst, int layer, int64_t part) {
  const int64_t src = a.table[n.parent * a.ld_table + n.full];
  if (src < 0 || src >= a.n_pages || src == dst) return;
  copy_item<false>(a.p0, a.p1, layer, src, dst, n.tail, part, a.parts);
}

// ---------------------------------------------------------------------------------------------
// update in one launch.  Every workgroup plans (prefix sums of the pages that slots ask for, and the free pages in
// ascending order); workgroup 0 writes the tables and counts refs in the LDS (integer sums: any order gives the same), the
// others copy tail pages, each 256 threads an item at a time.
struct UpdateLds {
  int count[kStepPages];
  uint16_t fresh[kStepPages];
  SlotPlan slot[kPlanThreads];
  uint16_t copies[kPlanThreads];
  int red[kPlanThreads / 64];
};
__global__ __launch_bounds__(kPlanThreads) void update_one_kernel(const PageArgs a) {
  extern __shared__ __align__(16) uint8_t lds_update[];
  UpdateLds& l = *(UpdateLds*)lds_update;
  const int tid = threadIdx.x, lane = tid & 63, per = per_wave(a.n_pages), base = wave_id() * per;
  int v[kBallots];
  uint64_t m[kBallots];
  const int mine = wave_pages<true>(a.refs, a.n_pages, base, per, v, m);
  SlotNeed n;
  bool ok = tid < a.S && slot_need(a, tid, n);
  int total, found, ncopy;
  const int ask = ok ? n.pages - n.full : 0;
  const int at = block_excl(ask, l.red, total);
  int free = waves_excl(mine, l.red, found);  // free pages below the wave's next 64
#pragma unroll
  for (int k = 0; k < kBallots; k++) {
    if (64 * k >= per) break;
    const int rank = free + lane_below(m[k]);
    if ((m[k] >> lane) & 1) l.fresh[rank] = (uint16_t)(base + 64 * k + lane);
    free += (int)__builtin_popcountll(m[k]);
  }
  ok = ok && at + ask <= found;
  const bool copy = ok && tail_rows(a, n) > 0;
  const int slot = block_excl(copy, l.red, ncopy);
  if (tid < a.S) l.slot[tid] = ok ? slot_plan(a, tid, at, n) : SlotPlan{-1};
  if (copy) l.copies[slot] = (uint16_t)tid;
  if (blockIdx.x > 0) {
    __syncthreads();
    const int64_t items = (int64_t)ncopy * a.items_per_copy * a.layers;
    constexpr int kGroups = kPlanThreads / kCopyThreads;
    for (int64_t i = (int64_t)(blockIdx.x - 1) * kGroups + tid / kCopyThreads; i < items; i += (int64_t)(gridDim.x - 1) * kGroups) {
      const int64_t cl = i / a.items_per_copy;
      const SlotPlan& p = l.slot[l.copies[cl / a.layers]];
      copy_tail(a, p, l.fresh[p.at], (int)(cl % a.layers), i - cl * a.items_per_copy);
    }
    return;
  }
  if (tid < a.S) {
    a.granted[tid] = ok;
    a.lens_out[tid] = ok ? n.next : a.lens[tid];
  }
#pragma unroll
  for (int k = 0; k < kBallots; k++)
    if (64 * k < per) l.count[base + 64 * k + lane] = v[k];
  __syncthreads();
  const int entries = a.S * a.M;
#pragma unroll 4
  for (int i = tid; i < entries; i += kPlanThreads) {
    const int s = (int)((uint32_t)i / (uint32_t)a.M), c = i - s * a.M;
    a.table_out[i] = slot_entry(a, s, c, l.slot[s], [&](int k) { return (int)l.fresh[k]; }, [&](int page, int by) {
      if (page >= 0 && page < a.n_pages) atomicAdd(&l.count[page], by);
    });
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kBallots; k++) {
    const int p = base + 64 * k + lane;
    if (64 * k < per && p < a.n_pages) a.refs_out[p] = l.count[p];
  }
}

// In two.  Workspace: [0] copies, [1 .. S] first fresh rank of a granted slot (-1: refused), [1 + S .. 1 + 2S] slots whose
// tail page is copied, then the fresh pages in rank order.
//
// Workgroup 0 plans; the others copy refs, which update_apply then counts up and down.
__global__ __launch_bounds__(kPlanThreads) void update_plan_kernel(const PageArgs a) {
  __shared__ int red[kPlanThreads / 64];
  __shared__ int ncopy;
  const int tid = threadIdx.x, lane = tid & 63;
  if (blockIdx.x > 0) {
    const int64_t i = (int64_t)(blockIdx.x - 1) * kPlanThreads + tid;
    if (i < a.n_pages) a.refs_out[i] = a.refs[i];
    return;
  }
  int32_t* rank = a.ws + 1;
  int32_t* copies = rank + a.S;
  int32_t* fresh = copies + a.S;
  if (tid == 0) ncopy = 0;
  int total = 0;
  for (int s0 = 0; s0 < a.S; s0 += kPlanThreads) {
    const int s = s0 + tid;
    SlotNeed n;
    const bool ok = s < a.S && slot_need(a, s, n);
    int sum;
    const int at = block_excl(ok ? n.pages - n.full : 0, red, sum);
    // (past 31 bits more pages are asked for than there are: refused)
    const int64_t first = (int64_t)total + at;
    if (s < a.S) rank[s] = ok && first <= a.n_pages ? (int)first : -1;
    total = (int)min((int64_t)total + sum, (int64_t)0x3fffffff);
  }
  int found = 0;
  for (int64_t step = 0; step < a.n_pages && found < total; step += kStepPages) {
    const int64_t base = step + wave_id() * kWavePages;
    int v[kBallots], sum;
    uint64_t m[kBallots];
    const int mine = wave_pages<true>(a.refs, a.n_pages, base, kWavePages, v, m);
    int free = found + waves_excl(mine, red, sum);
#pragma unroll
    for (int k = 0; k < kBallots; k++) {
      const int at = free + lane_below(m[k]);
      if (((m[k] >> lane) & 1) && at < total) fresh[at] = (int)(base + 64 * k + lane);
      free += (int)__builtin_popcountll(m[k]);
    }
    found += sum;
  }
  __syncthreads();
  for (int s = tid; s < a.S; s += kPlanThreads) {
    SlotNeed n;
    const int at = rank[s];
    const bool ok = at >= 0 && slot_need(a, s, n) && (int64_t)at + n.pages - n.full <= found;
    if (!ok) rank[s] = -1;
    a.granted[s] = ok;
    a.lens_out[s] = ok ? n.next : a.lens[s];
    if (ok && tail_rows(a, n) > 0) copies[atomicAdd(&ncopy, 1)] = s;
  }
  __syncthreads();
  if (tid == 0) a.ws[0] = ncopy;
}

// The first `row_blocks` workgroups write the table entries and count refs, the others copy tail pages, an item of
// kCopyChunk bytes at a time.
__global__ __launch_bounds__(kCopyThreads) void update_apply_kernel(const PageArgs a, int row_blocks) {
  const int32_t* rank = a.ws + 1;
  const int32_t* copies = rank + a.S;
  const int32_t* fresh = copies + a.S;
  if ((int)blockIdx.x < row_blocks) {
    const int64_t all = (int64_t)a.S * a.M;
    for (int64_t i = (int64_t)blockIdx.x * kCopyThreads + threadIdx.x; i < all; i += (int64_t)row_blocks * kCopyThreads) {
      const int s = (int)((uint32_t)i / (uint32_t)a.M), c = (int)((uint32_t)i - (uint32_t)s * (uint32_t)a.M);
      SlotNeed n;
      const int at = rank[s];
      if (at >= 0) slot_need(a, s, n);
      a.table_out[i] = slot_entry(a, s, c, at >= 0 ? slot_plan(a, s, at, n) : SlotPlan{-1}, [&](int k) { return fresh[k]; }, [&](int page, int by) {
        if (page >= 0 && page < a.n_pages) atomicAdd(a.refs_out + page, by);
      });
    }
    return;
  }
  const int64_t items = (int64_t)a.ws[0] * a.items_per_copy * a.layers;
  for (int64_t i = (int64_t)blockIdx.x - row_blocks; i < items; i += (int64_t)gridDim.x - row_blocks) {
    const int64_t cl = i / a.items_per_copy;
    const int s = copies[cl / a.layers];
    SlotNeed n;
    slot_need(a, s, n);
    copy_tail(a, slot_plan(a, s, rank[s], n), fresh[rank[s]], (int)(cl % a.layers), i - cl * a.items_per_copy);
  }
}

// ---------------------------------------------------------------------------------------------
// compact.  With L live pages, L0 of them below id L: a hole is a free page below L, its rank the free pages below it; a mover
// a live page from L on, its rank the live pages below it less L0; the mover of a rank goes to the hole of that rank.
//
// In one launch: every workgroup plans and copies its share of the pages, each 256 threads an item at a time;
// workgroup 0 writes refs, and the table's entries are spread over all.
struct CompactLds {
  uint16_t to[kStepPages];  // where a page's rows are afterwards (0xffff: not a live page)
  uint16_t holes[kStepPages / 2], movers[kStepPages / 2];
  int red[kPlanThreads / 64];
};
__global__ __launch_bounds__(kPlanThreads) void compact_one_kernel(const PageArgs a) {
  extern __shared__ __align__(16) uint8_t lds_compact[];
  CompactLds& l = *(CompactLds*)lds_compact;
  const int tid = threadIdx.x, lane = tid & 63, per = per_wave(a.n_pages), base = wave_id() * per;
  uint64_t m[kBallots];
  int live, low = 0, mine;
  {
    int v[kBallots];
    mine = wave_pages<false>(a.refs, a.n_pages, base, per, v, m);
  }
  const int before = waves_excl(mine, l.red, live);
#pragma unroll
  for (int k = 0; k < kBallots; k++)
    if (64 * k < per) low += bits_below(m[k], live - (base + 64 * k));
  int l0;
  waves_excl(low, l.red, l0);
  int below = before;  // live pages below the wave's next 64
#pragma unroll
  for (int k = 0; k < kBallots; k++) {
    if (64 * k >= per) break;
    const int p = base + 64 * k + lane, rank = below + lane_below(m[k]);
    const bool is = (m[k] >> lane) & 1;
    l.to[p] = (uint16_t)(is ? p : 0xffff);
    if (is && p >= live) l.movers[rank - l0] = (uint16_t)p;
    if (!is && p < live) l.holes[p - rank] = (uint16_t)p;
    below += (int)__builtin_popcountll(m[k]);
  }
  const int moved = live - l0;
  __syncthreads();
  for (int i = tid; i < moved; i += kPlanThreads) l.to[l.movers[i]] = l.holes[i];
  const int64_t items = (int64_t)moved * a.items_per_copy * a.layers;
  constexpr int kGroups = kPlanThreads / kCopyThreads;
  for (int64_t i = (int64_t)blockIdx.x * kGroups + tid / kCopyThreads; i < items; i += (int64_t)gridDim.x * kGroups) {
    const int64_t cl = i / a.items_per_copy, at = cl / a.layers;
    copy_item<true>(a.p0, a.p1, (int)(cl % a.layers), l.movers[at], l.holes[at], a.P, i - cl * a.items_per_copy, a.parts);
  }
  __syncthreads();
  const int64_t n = (int64_t)a.S * a.M;
  for (int64_t i = (int64_t)blockIdx.x * kPlanThreads + tid; i < n; i += (int64_t)gridDim.x * kPlanThreads) {
    const uint32_t s = (uint32_t)i / (uint32_t)a.M, c = (uint32_t)i - s * (uint32_t)a.M;
    const int page = a.table[s * a.ld_table + c];
    const int to = page >= 0 && page < a.n_pages ? l.to[page] : 0xffff;
    a.table_out[i] = to == 0xffff ? -1 : to;
  }
  if (blockIdx.x > 0) return;
  if (tid == 0) a.live[0] = live;
  below = before;
#pragma unroll
  for (int k = 0; k < kBallots; k++) {
    if (64 * k >= per) break;
    const int p = base + 64 * k + lane, rank = below + lane_below(m[k]);
    below += (int)__builtin_popcountll(m[k]);
    if (p >= a.n_pages) continue;
    const bool is = (m[k] >> lane) & 1;
    const int r = a.refs[!is && p < live ? l.movers[p - rank] : p];
    a.refs_out[p] = is && p >= live ? 0 : r;
  }
}

// In two.  Workspace: [0] live pages, [1] moved pages, then rank [n_pages] (a moving page's or a hole's),
// holes [n_pages], movers [n_pages].
__global__ __launch_bounds__(kPlanThreads) void compact_plan_kernel(const PageArgs a) {
  __shared__ int red[kPlanThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63;
  int32_t* rank = a.ws + 2;
  int32_t* holes = rank + a.n_pages;
  int32_t* movers = holes + a.n_pages;
  int v[kBallots], mine = 0, live;
  uint64_t m[kBallots];
  for (int64_t step = 0; step < a.n_pages; step += kStepPages)
    mine += wave_pages<false>(a.refs, a.n_pages, step + wave_id() * kWavePages, kWavePages, v, m);
  waves_excl(mine, red, live);
  int before = 0, l0 = 0;  // live pages of the steps so far; of those, below `live`
  for (int64_t step = 0; step < a.n_pages; step += kStepPages) {
    const int64_t base = step + wave_id() * kWavePages;
    const int here = wave_pages<false>(a.refs, a.n_pages, base, kWavePages, v, m);
    int sum, lsum, low = 0;
    int below = before + waves_excl(here, red, sum);
#pragma unroll
    for (int k = 0; k < kBallots; k++) low += bits_below(m[k], live - (base + 64 * k));
    waves_excl(low, red, lsum);
    before += sum;
    l0 += lsum;  // (all of L0 where the step has a page past `live`)
#pragma unroll
    for (int k = 0; k < kBallots; k++) {
      const int64_t p = base + 64 * k + lane;
      const int at = below + lane_below(m[k]);
      below += (int)__builtin_popcountll(m[k]);
      if (p >= a.n_pages) continue;
      if ((m[k] >> lane) & 1) {
        if (p >= live) {
          rank[p] = at - l0;
          movers[at - l0] = (int)p;
        }
      } else if (p < live) {
        rank[p] = (int)p - at;
        holes[(int)p - at] = (int)p;
      }
    }
  }
  if (tid == 0) {
    a.ws[0] = live;
    a.ws[1] = live - l0;
    a.live[0] = live;
  }
}

__global__ __launch_bounds__(kCopyThreads) void compact_apply_kernel(const PageArgs a, int row_blocks) {
  const int live = a.ws[0];
  const int32_t* rank = a.ws + 2;
  const int32_t* holes = rank + a.n_pages;
  const int32_t* movers = holes + a.n_pages;
  if ((int)blockIdx.x < row_blocks) {
    const int64_t n = (int64_t)a.S * a.M, step = (int64_t)row_blocks * kCopyThreads;
    const int64_t t0 = (int64_t)blockIdx.x * kCopyThreads + threadIdx.x;
    for (int64_t i = t0; i < n; i += step) {
      const uint32_t s = (uint32_t)i / (uint32_t)a.M, c = (uint32_t)i - s * (uint32_t)a.M;
      const int page = a.table[s * a.ld_table + c];
      int to = -1;
      if (page >= 0 && page < a.n_pages && a.refs[page] > 0) to = page < live ? page : holes[rank[page]];
      a.table_out[i] = to;
    }
    for (int64_t i = t0; i < a.n_pages; i += step) {
      const int r = a.refs[i];
      a.refs_out[i] = i < live ? (r > 0 ? r : a.refs[movers[rank[i]]]) : (r > 0 ? 0 : r);
    }
    return;
  }
  const int64_t items = (int64_t)a.ws[1] * a.items_per_copy * a.layers;
  for (int64_t i = (int64_t)blockIdx.x - row_blocks; i < items; i += (int64_t)gridDim.x - row_blocks) {
    const int64_t cl = i / a.items_per_copy, part = i - cl * a.items_per_copy;
    const int64_t m = cl / a.layers;
    copy_item<true>(a.p0, a.p1, (int)(cl % a.layers), movers[m], holes[m], a.P, part, a.parts);
  }
}

int check_pages(const PageArgs& a, int64_t S, int64_t M, int64_t n_pages, int64_t P, int64_t layers) {
  if (!a.table || !a.refs || !a.table_out || !a.refs_out || !a.p0.base) return SMLA_E_NULL;
  if (S <= 0 || M <= 0 || n_pages <= 0 || P <= 0 || layers <= 0 || a.p0.row_bytes <= 0 || a.ld_table < M)
    return SMLA_E_SHAPE;
  if (S * M > 0x7fffffff || n_pages > 0x3fffffff || P > 0x3fffffff || layers > 0xffff) return SMLA_E_RANGE;
  if (a.p1.base && a.p1.row_bytes <= 0) return SMLA_E_SHAPE;
  if (a.table_out == a.table || a.refs_out == a.refs) return SMLA_E_UNSUPPORTED;
  return SMLA_OK;
}

PageArgs page_args(const int32_t* table, int64_t ld_table, int64_t S, int64_t M, const int32_t* refs, int64_t n_pages,
                   int64_t P, int32_t* table_out, int32_t* refs_out, void* pages, int64_t layers, int64_t layer_bytes,
                   int64_t row_bytes, void* scales, int64_t scale_layer_bytes, int64_t scale_row_bytes, void* ws) {
  PageArgs a{};
  a.table = table;
  a.refs = refs;
  a.ld_table = ld_table;
  a.S = (int)S;
  a.M = (int)M;
  a.n_pages = (int)n_pages;
  a.P = (int)P;
  a.layers = (int)layers;
  a.table_out = table_out;
  a.refs_out = refs_out;
  a.p0 = Pool{(uint8_t*)pages, layer_bytes, P * row_bytes, row_bytes};
  a.p1 = Pool{(uint8_t*)scales, scale_layer_bytes, P * scale_row_bytes, scale_row_bytes};
  a.parts = (P * row_bytes + kCopyChunk - 1) / kCopyChunk;
  a.items_per_copy = a.parts + (scales ? 1 : 0);
  a.ws = (int32_t*)ws;
  return a;
}

// workgroups of the table part and of the copies: a few per compute unit, each walking its share
int row_blocks(int64_t n) {
  const int64_t want = (n + kCopyThreads - 1) / kCopyThreads, most = 2 * smla_num_cus();
  return (int)(want < most ? want : most);
}
int copy_blocks(const PageArgs& a, int64_t entries) {
  const int64_t want = entries * a.items_per_copy * a.layers, most = 8 * smla_num_cus();
  return (int)(want < most ? want : most);
}
// workgroups of kPlanThreads for the copies of a call in one launch
int one_blocks(const PageArgs& a, int64_t entries, int64_t most) {
  const int64_t groups = kPlanThreads / kCopyThreads, want = (entries * a.items_per_copy * a.layers + groups - 1) / groups;
  return (int)(want < most ? want : most);
}
bool update_in_one(int64_t S, int64_t M, int64_t n_pages) {
  return S <= kPlanThreads && n_pages <= kStepPages && S * M <= kOneEntries;
}
bool compact_in_one(int64_t n_pages) { return n_pages <= kStepPages; }
bool has_workspace(const void* ws, size_t bytes, size_t need) {
  return need == 0 || (ws && ((uintptr_t)ws & 3) == 0 && bytes >= need);
}

}  // namespace

extern "C" size_t smla_update_pages_workspace(int64_t S, int64_t M, int64_t n_pages) {
  return S > 0 && M > 0 && n_pages > 0 && !update_in_one(S, M, n_pages) ? (size_t)(1 + 2 * S + n_pages) * 4 : 0;
}

extern "C" int smla_update_pages(const int32_t* table, int64_t ld_table, int64_t S, int64_t M, const int32_t* lens,
                                 const int32_t* refs, int64_t n_pages, int64_t P, const int32_t* parent,
                                 const int32_t* grow, int32_t* table_out, int32_t* lens_out, int32_t* refs_out,
                                 int32_t* granted, void* pages, int64_t layers, int64_t layer_bytes, int64_t row_bytes,
                                 void* scales, int64_t scale_layer_bytes, int64_t scale_row_bytes, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  if (!lens || !parent || !grow || !lens_out || !granted) return SMLA_E_NULL;
  PageArgs a = page_args(table, ld_table, S, M, refs, n_pages, P, table_out, refs_out, pages, layers, layer_bytes,
                         row_bytes, scales, scale_layer_bytes, scale_row_bytes, workspace);
  if (int rc = check_pages(a, S, M, n_pages, P, layers); rc != 0) return rc;
  if (lens_out == lens) return SMLA_E_UNSUPPORTED;
  if (!has_workspace(workspace, workspace_bytes, smla_update_pages_workspace(S, M, n_pages))) return SMLA_E_WORKSPACE;
  a.lens = lens;
  a.parent = parent;
  a.grow = grow;
  a.lens_out = lens_out;
  a.granted = granted;
  const hipStream_t st = (hipStream_t)stream;
  if (update_in_one(S, M, n_pages)) {
    static std::atomic<uint64_t> lds_attr{0};
    if (hipError_t e = smla_set_dynamic_lds((const void*)update_one_kernel, sizeof(UpdateLds), lds_attr); e != hipSuccess)
      return (int)e;
    hipLaunchKernelGGL(update_one_kernel, dim3((unsigned)(1 + one_blocks(a, S, smla_num_cus()))), dim3(kPlanThreads),
                       sizeof(UpdateLds), st, a);
    SMLA_HIP_CHECK_LAUNCH();
    return SMLA_OK;
  }
  hipLaunchKernelGGL(update_plan_kernel, dim3((unsigned)(1 + (n_pages + kPlanThreads - 1) / kPlanThreads)),
                     dim3(kPlanThreads), 0, st, a);
  SMLA_HIP_CHECK_LAUNCH();
  const int rb = row_blocks(S * M);
  hipLaunchKernelGGL(update_apply_kernel, dim3((unsigned)(rb + copy_blocks(a, S))), dim3(kCopyThreads), 0, st, a, rb);
  SMLA_HIP_CHECK_LAUNCH();
  return SMLA_OK;
}

extern "C" size_t smla_compact_pages_workspace(int64_t n_pages) {
  return n_pages > 0 && !compact_in_one(n_pages) ? (size_t)(2 + 3 * n_pages) * 4 : 0;
}

extern "C" int smla_compact_pages(const int32_t* table, int64_t ld_table, int64_t S, int64_t M, const int32_t* refs,
                                  int64_t n_pages, int64_t P, int32_t* table_out, int32_t* refs_out, int32_t* live,
                                  void* pages, int64_t layers, int64_t layer_bytes, int64_t row_bytes, void* scales,
                                  int64_t scale_layer_bytes, int64_t scale_row_bytes, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  if (!live) return SMLA_E_NULL;
  PageArgs a = page_args(table, ld_table, S, M, refs, n_pages, P, table_out, refs_out, pages, layers, layer_bytes,
                         row_bytes, scales, scale_layer_bytes, scale_row_bytes, workspace);
  if (int rc = check_pages(a, S, M, n_pages, P, layers); rc != 0) return rc;
  if (!has_workspace(workspace, workspace_bytes, smla_compact_pages_workspace(n_pages))) return SMLA_E_WORKSPACE;
  a.live = live;
  const hipStream_t st = (hipStream_t)stream;
  if (compact_in_one(n_pages)) {
    static std::atomic<uint64_t> lds_attr{0};
    if (hipError_t e = smla_set_dynamic_lds((const void*)compact_one_kernel, sizeof(CompactLds), lds_attr); e != hipSuccess)
      return (int)e;
    hipLaunchKernelGGL(compact_one_kernel, dim3((unsigned)(1 + one_blocks(a, n_pages / 2, smla_num_cus() - 1))),
                       dim3(kPlanThreads), sizeof(CompactLds), st, a);
    SMLA_HIP_CHECK_LAUNCH();
    return SMLA_OK;
  }
  hipLaunchKernelGGL(compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, a);
  SMLA_HIP_CHECK_LAUNCH();
  const int rb = row_blocks(S * M > n_pages ? S * M : n_pages);
  hipLaunchKernelGGL(compact_apply_kernel, dim3((unsigned)(rb + copy_blocks(a, (n_pages + 1) / 2))),
                     dim3(kCopyThreads), 0, st, a, rb);
  SMLA_HIP_CHECK_LAUNCH();
  return SMLA_OK;
}

extern "C" int smla_paged_append_granted(const void* q, int64_t ldq, const void* kv, int64_t ldkv, int x_dtype, int64_t T,
                                         int64_t H, int64_t D, int64_t norm_dims, const float* q_w, const float* kv_w,
                                         const float* cos_t, const float* sin_t, int64_t n_pos, int64_t rd, float eps,
                                         int sim, int flags, void* q_out, void* pages, int page_dtype, float* scales,
                                         int64_t n_pages, int64_t P, const int32_t* table, int64_t ld_table, int64_t cols,
                                         const int32_t* lens, const int32_t* cu, const int32_t* granted, int64_t B,
                                         void* stream) {
  if (!kv || !pages || !table || !lens || !cu || (H > 0 && (!q || !q_out)) || (rd > 0 && (!cos_t || !sin_t)))
    return SMLA_E_NULL;
  if (T < 0 || H < 0 || D <= 0 || B <= 0 || n_pages <= 0 || P <= 0 || cols <= 0 || ld_table < cols || rd < 0 ||
      rd > D || norm_dims < 0 || norm_dims > D || ldkv < D || (H > 0 && ldq < H * D) || (rd > 0 && n_pos <= 0))
    return SMLA_E_SHAPE;
  if (x_dtype != SMLA_F32 && x_dtype != SMLA_BF16) return SMLA_E_DTYPE;
  if (page_dtype != SMLA_BF16 && page_dtype != SMLA_FP8_E4M3) return SMLA_E_DTYPE;
  if (page_dtype == SMLA_FP8_E4M3 && !scales) return SMLA_E_NULL;
  if ((flags & ~(SMLA_PAGED_NORM_Q | SMLA_PAGED_NORM_KV | SMLA_PAGED_FILL)) != 0) return SMLA_E_RANGE;
  if ((flags & (SMLA_PAGED_NORM_Q | SMLA_PAGED_NORM_KV)) && norm_dims == 0) return SMLA_E_SHAPE;
  if (sim != SMLA_SIM_NONE && (sim != SMLA_SIM_FP8 || page_dtype != SMLA_BF16)) return SMLA_E_UNSUPPORTED;
  if (D % 64 != 0 || D > 1024 || norm_dims % 4 != 0 || rd % 4 != 0 || (sim == SMLA_SIM_FP8 && rd % 64 != 0))
    return SMLA_E_UNSUPPORTED;
  // a lane reads four channels at a time (two boundaries of a rotation pair never part)
  const uintptr_t xa = x_dtype == SMLA_F32 ? 15 : 7;
  if (((uintptr_t)kv & xa) || ldkv % 4 || ((uintptr_t)pages & 7) || ((uintptr_t)q & xa) || (H > 0 && ldq % 4) ||
      ((uintptr_t)q_out & 7))
    return SMLA_E_UNSUPPORTED;
  if (T > 0x7fffffff || B > 0x7fffffff || n_pages > 0x3fffffff || P > 0x3fffffff || cols > 0x7fffffff ||
      T * (H + 1) > 0x7fffffff)
    return SMLA_E_RANGE;
  if (T == 0) return SMLA_OK;
  // rows of q and kv are read while others of q_out are written; a row is read whole before it is written, so q itself
  // (dense, bf16) may be q_out
  const uintptr_t es = x_dtype == SMLA_F32 ? 4 : 2, o0 = (uintptr_t)q_out, o1 = o0 + (uintptr_t)T * H * D * 2;
  auto over = [&](const void* p, int64_t ld, int64_t w) {
    return o0 < (uintptr_t)p + ((uintptr_t)(T - 1) * ld + w) * es && (uintptr_t)p < o1;
  };
  const bool same = q == q_out && x_dtype == SMLA_BF16 && (T == 1 || ldq == H * D);
  if (H > 0 && ((!same && over(q, ldq, H * D)) || over(kv, ldkv, D))) return SMLA_E_UNSUPPORTED;
  AppendArgs a{};
  a.q = q;
  a.kv = kv;
  a.ldq = ldq;
  a.ldkv = ldkv;
  a.T = (uint32_t)T;
  a.H = (uint32_t)H;
  a.rows_per_tok = (uint32_t)H + 1;
  a.D = (int)D;
  a.norm_dims = (int)norm_dims;
  a.rd = (int)rd;
  a.flags = flags;
  a.sim = sim;
  a.page_dtype = page_dtype;
  a.q_w = q_w;
  a.kv_w = kv_w;
  a.cos_t = cos_t;
  a.sin_t = sin_t;
  a.n_pos = n_pos;
  a.eps = eps;
  a.q_out = (uint16_t*)q_out;
  a.pages = pages;
  a.scales = scales;
  a.n_pages = (int)n_pages;
  a.P = (int)P;
  a.cols = (int)cols;
  a.B = (int)B;
  a.ld_table = ld_table;
  a.table = table;
  a.lens = lens;
  a.cu = cu;
  a.granted = granted;
  const dim3 grid((unsigned)((T * (H + 1) + 3) / 4)), block(256);
  const hipStream_t st = (hipStream_t)stream;
#define SMLA_APPEND(X, N) hipLaunchKernelGGL((paged_append_kernel<X, N>), grid, block, 0, st, a)
#define SMLA_APPEND_D(X)                 \
  do {                                   \
    if (D <= 512) SMLA_APPEND(X, 2);      \
    else if (D <= 768) SMLA_APPEND(X, 3); \
    else SMLA_APPEND(X, 4);               \
  } while (0)
  if (x_dtype == SMLA_F32) SMLA_APPEND_D(SMLA_F32);
  else SMLA_APPEND_D(SMLA_BF16);
#undef SMLA_APPEND_D
#undef SMLA_APPEND
  SMLA_HIP_CHECK_LAUNCH();
  return SMLA_OK;
}

extern "C" int smla_paged_append(const void* q, int64_t ldq, const void* kv, int64_t ldkv, int x_dtype, int64_t T,
                                 int64_t H, int64_t D, int64_t norm_dims, const float* q_w, const float* kv_w,
                                 const float* cos_t, const float* sin_t, int64_t n_pos, int64_t rd, float eps, int sim,
                                 int flags, void* q_out, void* pages, int page_dtype, float* scales, int64_t n_pages,
                                 int64_t P, const int32_t* table, int64_t ld_table, int64_t cols, const int32_t* lens,
                                 const int32_t* cu, int64_t B, void* stream) {
  return smla_paged_append_granted(q, ldq, kv, ldkv, x_dtype, T, H, D, norm_dims, q_w, kv_w, cos_t, sin_t, n_pos, rd, eps,
                                   sim, flags, q_out, pages, page_dtype, scales, n_pages, P, table, ld_table, cols, lens,
                                   cu, nullptr, B, stream);
}
