// The K loop of the tiled products with 4-bit or bf16 weights (experts.hip): one workgroup's BM x BN tile of
// x . W^T, x bf16 rows anywhere, W rows of codes with scales or of bf16, sums in fp32 by v_mfma_f32_32x32x16_bf16.
//
// Operands go HBM -> LDS by copies of 1 KB a wave into a ring of D stages of KB k: 128 k of 4-bit weights are 64 bytes
// a row (one b128 read a lane is 32 k: the operands of four products), 64 k of bf16 are 128.  Codes stay codes in LDS,
// a quarter of the bytes to copy and to read, and become bf16 in registers between the products (four 4-cycle
// conversions a 32 x 16 operand, one product's 32 cycles take it in).  For a lane to hold 32 consecutive k of a weight
// row, a product's k are not 16 neighbours: lane half h of product j of a 64-k group g takes k 64 g + 32 h + 8 j .. + 7,
// of both operands.
//
// A copy lands contiguously, so rows cannot be padded: chunks of 16 bytes are permuted within a row so that 16
// consecutive rows' reads of one column fall in distinct banks (swx, sww).
//
// What bounds it is issue, as in gemm_tile.h, whose order of a step it keeps: the next sub-step's reads and conversions
// and the copies of a later step stand between the products of this one, the one barrier of a step before its last
// sub-step, whose operands are in registers by then.
//
// K that is no multiple of KB: the range is padded in front to whole steps.  The first step's chunks that do not exist
// are read from the row's first ones and zeroed in LDS before use.
#pragma once

#include "fp4.h"
#include "gemm_tile.h"

namespace smla_tile {

using smla_attn::lds_barrier;
using smla_attn::lds_u32x4_t;
using smla_attn::lds_u8_t;
using smla_attn::wait_vm;
using smla_gemm::Int;

constexpr int kFp4 = 0, kBf16 = 1;

template <int WT_, int BM_, int BN_, int WM_, int WN_, int D_, int KB_>
struct Tile {
  static constexpr int WT = WT_, BM = BM_, BN = BN_, WM = WM_, WN = WN_, D = D_, KB = KB_, SUB = KB / 16;
  static constexpr int XROW = 2 * KB, WROW = WT == kFp4 ? KB / 2 : 2 * KB;  // bytes of a row per step
  static constexpr int XC = XROW / 16, WC = WROW / 16;                        // chunks
  static constexpr int NWN = BN / WN, NW = (BM / WM) * NWN, MB = WM / 32, NB = WN / 32;
  static constexpr int XB = BM * XROW, WB = BN * WROW, STAGE = XB + WB;
  static constexpr int SG = WT == kFp4 ? BN * 16 : 0;  // a group of scales, 512 k
  static constexpr int CX = XB / 1024 / NW, CW = WB / 1024 / NW, CP = CX + CW;  // copies a wave and step
  static constexpr int GS = WT == kFp4 ? 512 / KB : 1, CS = WT == kFp4 ? 4 / GS : 0, CT = CP + CS;  // steps of a group of scales
  static constexpr int LDS = D * STAGE + 3 * SG;
  static constexpr int THREADS = 64 * NW;
  static_assert(CX * NW * 1024 == XB && CW * NW * 1024 == WB && BN % 64 == 0 && (WN == 64 || (WN == 128 && BM == 2 * WM)), "whole copies per wave");
  static_assert((WT == kFp4 ? KB == 128 || KB == 256 : KB == 64) && D >= 2, "a step");
  static __device__ int swx(int r) { return XROW >= 256 ? r & 15 : (r >> 1) & 7; }
  static __device__ int sww(int r) { return WROW == 64 ? (r >> 2) & 3 : (r >> 1) & 7; }
};

// 4-byte copy for every lane (lane l lands at lds_dst + 4 l), addresses as dma16_s (the s_nop: a base that a vector
// instruction has just written, v_readfirstlane, is read five wait states later at the earliest)
__device__ inline void dma4_s(const uint8_t* base, uint32_t off, uint32_t lds_dst) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dword %1, %2" ::"s"(lds_dst), "v"(off), "s"(base) : "memory", "m0");
}

// a value that every lane of the wave has, in a scalar register (the copies' addresses need one)
__device__ inline const uint8_t* uniform(const uint8_t* p) {
  const uint64_t v = (uint64_t)p;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
  return (const uint8_t*)((uint64_t)hi << 32 | lo);
}

// What a tile multiplies.  x: row r of the tile at x + xoff(r); w[half]: tile row r is row wrow(r) of half whalf(r),
// ldw bytes apart; scales likewise, lds bytes apart, 4 a step.  All point at the first (padded) step.
struct Source {
  const uint8_t* x;
  const uint8_t* w[2];
  const uint8_t* s[2];
  uint32_t ldw, lds;
  int pad;  // k that the first step lacks
};

// acc[mb][nb], mb < MBV, of wave (wm, wn) = (wave / NWN, wave % NWN): accumulator register r is row WM wm + 32 mb +
// 8 (r / 4) + 4 (lane / 32) + r mod 4 of x, row WN wn + 32 nb + lane mod 32 of w, over steps >= 1 steps.  MBV differs between
// the waves of a tile with fewer rows; all take part in the copies.
template <class L, int MBV, class XO, class WR, class WH>
__device__ __attribute__((always_inline)) inline void tile_loop(lds_u8_t* lds, const Source& src, int steps, XO&& xoff, WR&& wrow,
                                                                WH&& whalf, f32x16_t (&acc)[MBV > 0 ? MBV : 1][L::NB]) {
  constexpr int NB = L::NB, NM = MBV * NB, D = L::D, SUB = L::SUB, CT = L::CT;
  const uint32_t lds_base = (uint32_t)(uintptr_t)lds;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / L::NWN, wn = wave % L::NWN;
  const int nk = __builtin_amdgcn_readfirstlane(steps);
  uint32_t off[L::CP], off0[L::CP];  // of every step but the padded one
  const uint8_t* wb[L::CW];
  const uint8_t* xb = uniform(src.x);
#pragma unroll
  for (int i = 0; i < L::CX; i++) {
    const int r = (wave * L::CX + i) * (64 / L::XC) + lane / L::XC, c = (lane % L::XC) ^ L::swx(r);
    const uint32_t row = xoff(r);
    off[i] = row + 16 * c;
    off0[i] = row + max(16 * c, 2 * src.pad);
  }
#pragma unroll
  for (int i = 0; i < L::CW; i++) {
    const int r0 = (wave * L::CW + i) * (64 / L::WC), r = r0 + lane / L::WC, c = (lane % L::WC) ^ L::sww(r);
    const uint32_t row = (uint32_t)wrow(r) * src.ldw;
    wb[i] = uniform(whalf(r0) ? src.w[1] : src.w[0]);
    off[L::CX + i] = row + 16 * c;
    off0[L::CX + i] = row + max(16 * c, L::WT == kFp4 ? src.pad / 2 : 2 * src.pad);
  }
  // scales: 512 k of a row are 16 bytes (a step's four alone, 64 rows a request, took as many requests as all the
  // weights).  With a step's copies a wave requests those of 16 (KB = 256: 32) of its rows for the group behind the
  // step's, so that a group is there when its first step is; three groups in LDS.
  const int su = L::WN == 64 ? 64 * wn : 64 * (2 * wn + wm);
  uint32_t so0 = (uint32_t)wrow(su + (lane >> 2)) * src.lds, so1 = (uint32_t)wrow(su + 16 + (lane >> 2)) * src.lds,
           so2 = (uint32_t)wrow(su + 32 + (lane >> 2)) * src.lds, so3 = (uint32_t)wrow(su + 48 + (lane >> 2)) * src.lds;
  asm volatile("" : "+v"(so0), "+v"(so1), "+v"(so2), "+v"(so3));  // (four registers, not an array in scratch memory)
  const uint8_t* sb[2] = {uniform(L::WT == kFp4 ? src.s[0] : src.x), uniform(L::WT == kFp4 ? src.s[1] : src.x)};
  const uint32_t sl = lds_base + D * L::STAGE + 16 * su;
  const int lack = src.pad / 128, words = nk * (L::KB / 128) - lack;  // a row's groups of 128 k: those of the pad are not there
  auto copy_scales = [&](int part, int of) __attribute__((always_inline)) {
    const int j = __builtin_amdgcn_readfirstlane(part), group = __builtin_amdgcn_readfirstlane(of);  // (scalar registers for the copy)
    const int w = min(max(4 * group + (lane & 3) - lack, 0), words - 1);
    const uint32_t o = (j == 0 ? so0 : j == 1 ? so1 : j == 2 ? so2 : so3) + 4 * w;
    dma4_s(whalf(su + 16 * j) ? sb[1] : sb[0], o, sl + (group % 3) * L::SG + 256 * j);
  };
  auto copy_to = [&](int ks, int stage, int i, bool head) __attribute__((always_inline)) {
    const uint32_t st = lds_base + stage * L::STAGE;
    if (i < L::CP) {
      const uint8_t* base = i < L::CX ? xb + (int64_t)ks * L::XROW : wb[i < L::CX ? 0 : i - L::CX] + (int64_t)ks * L::WROW;
      const int q = i < L::CX ? wave * L::CX + i : L::XB / 1024 + wave * L::CW + i - L::CX;
      smla_gemm::dma16_s(base, head ? off0[i] : off[i], st + q * 1024);
    } else {
      copy_scales(ks % L::GS * L::CS + i - L::CP, ks / L::GS + 1);
    }
  };
  auto copy = [&](int ks, int i) __attribute__((always_inline)) { copy_to(ks, ks % D, i, false); };
  // operands: a of this lane's row, chunks as above; raw: 32 codes and their scale, or nothing
  const int r32 = lane & 31, h = lane >> 5, sx = L::swx(r32), sw = L::sww(r32);
  const uint32_t xrow = (L::WM * wm + r32) * L::XROW, wrw = L::XB + (L::WN * wn + r32) * L::WROW,
                 srow = D * L::STAGE + (L::WN * wn + r32) * 16;
  bf16x8_t a[2][MBV > 0 ? MBV : 1], b[2][NB];
  u32x4_t raw[2][NB];
  uint32_t rs[2 * NB];  // a step's scale bytes, of its first 128 k and of its second
  auto read_a = [&](int ks, int kk, int m) __attribute__((always_inline)) {
    const lds_u8_t* p = lds + (ks % D) * L::STAGE + 16 * ((8 * (kk / 4) + 4 * h + kk % 4) ^ sx) + xrow + 32 * L::XROW * m;
    a[kk & 1][m] = as_bf16x8(*(const lds_u32x4_t*)p);
  };
  auto read_b = [&](int ks, int kk, int n) __attribute__((always_inline)) {  // kk: the first sub-step of a 64-k group, or any of bf16
    const lds_u8_t* st = lds + (ks % D) * L::STAGE;
    if constexpr (L::WT == kFp4) {
      const int g = kk / 4;
      raw[g & 1][n] = *(const lds_u32x4_t*)(st + wrw + 32 * L::WROW * n + 16 * ((2 * g + h) ^ sw));
      if (g == 0) {
        const lds_u8_t* at = lds + srow + 512 * n + (ks / L::GS % 3) * L::SG + ks % L::GS * (16 / L::GS);
        rs[n] = *(const smla_attn::lds_i32_t*)at;
        if constexpr (L::KB == 256) rs[NB + n] = *(const smla_attn::lds_i32_t*)(at + 4);
      }
    } else {
      b[kk & 1][n] = as_bf16x8(*(const lds_u32x4_t*)(st + wrw + 32 * L::WROW * n + 16 * ((4 * h + kk) ^ sw)));
    }
  };
  auto convert = [&](int kk, int n) __attribute__((always_inline)) {
    if constexpr (L::WT == kFp4)
      b[kk & 1][n] = smla_fp4::to_bf16(raw[(kk / 4) & 1][n][kk % 4], smla_fp4::scale_of(rs[kk / 8 * NB + n] >> (8 * h + kk / 4 % 2 * 16) & 255));
  };
  // the products of sub-step kk, with what comes between them: the operands of sub-step (ns, nkk) (nkk < 0: none), raw
  // codes of group (gs, gk) (gk < 0: none), copies i0 .. i1-1 of step `is`
  auto sub = [&](auto kk_, int ns, auto nkk_, int gs, auto gk_, int is, auto i0_, auto i1_) __attribute__((always_inline)) {
    constexpr int kk = decltype(kk_)::value, nkk = decltype(nkk_)::value, gk = decltype(gk_)::value;
    constexpr int i0 = decltype(i0_)::value, i1 = decltype(i1_)::value;
    constexpr int RB = NM > 0 && (L::WT == kFp4 ? gk : nkk) >= 0 ? NB : 0, RA = nkk >= 0 ? MBV : 0, NR = RB + RA;
    constexpr int SL = NM > 0 ? NM : 1, RPM = (NR + SL - 1) / SL;
#pragma unroll
    for (int j = 0; j < SL; j++) {
#pragma unroll
      for (int e = j * RPM; e < (j + 1) * RPM && e < NR; e++) {
        if (e < RB) read_b(L::WT == kFp4 ? gs : ns, L::WT == kFp4 ? gk : nkk, e);
        else read_a(ns, nkk, e - RB);
      }
      if constexpr (NM > 0) {
        const int m = j / NB, n = j % NB;
        acc[m][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[kk & 1][m], b[kk & 1][n], acc[m][n], 0, 0, 0);
      }
#pragma unroll
      for (int e = i0 + j * (i1 - i0) / SL; e < i0 + (j + 1) * (i1 - i0) / SL; e++) copy(is, e);
      if constexpr (nkk >= 0 && NM > 0) {
        if (SL < NB || j >= SL - NB) {
#pragma unroll
          for (int n = 0; n < NB; n++)
            if (SL < NB ? j == SL - 1 : n == j - (SL - NB)) convert(nkk, n);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // copy i of a step goes out in part i NSP / CT of them: part 0 in sub-step SUB - 1, part p in sub-step p - 1 of the next step
  constexpr int NSP = SUB >= 8 ? SUB / 2 : 4, C0 = CT / NSP;
  // step ks: MORE: the rest of step ks + D - 1's copies goes out; FIRST: the first part of step ks + D's; NEXT: a step follows
  auto step = [&](int ks, auto more_, auto first_, auto next_) __attribute__((always_inline)) {
    constexpr int more = decltype(more_)::value, first = decltype(first_)::value, next = decltype(next_)::value;
    auto subs = [&](auto self, auto kk_) __attribute__((always_inline)) {
      constexpr int kk = decltype(kk_)::value, p = kk + 1;
      if constexpr (kk < SUB - 1) {
        constexpr int i0 = more && p < NSP ? p * CT / NSP : 0, i1 = more && p < NSP ? (p + 1) * CT / NSP : 0;
        sub(Int<kk>{}, ks, Int<kk + 1>{}, ks, Int<kk % 4 == 0 && kk + 4 < SUB ? kk + 4 : -1>{}, ks + D - 1, Int<i0>{}, Int<i1>{});
        self(self, Int<kk + 1>{});
      }
    };
    subs(subs, Int<0>{});
    if constexpr (next) {
      wait_vm(more ? (D - 2) * CT : 0);  // this wave's copies of step ks + 1
      lds_barrier();                      // everyone's; and step ks is in every wave's registers
      sub(Int<SUB - 1>{}, ks + 1, Int<0>{}, ks + 1, Int<0>{}, ks + D, Int<0>{}, Int<first ? C0 : 0>{});
    } else {
      sub(Int<SUB - 1>{}, 0, Int<-1>{}, 0, Int<-1>{}, 0, Int<0>{}, Int<0>{});
    }
  };
#pragma unroll
  for (int m = 0; m < MBV; m++)
#pragma unroll
    for (int n = 0; n < NB; n++)
#pragma unroll
      for (int r = 0; r < 16; r++) acc[m][n][r] = 0.f;
#pragma unroll
  for (int j = 0; j < (L::WT == kFp4 ? 4 : 0); j++) copy_scales(j, 0);
#pragma unroll
  for (int s = 0; s < D; s++)
#pragma unroll
    for (int i = 0; i < (s < D - 1 ? CT : C0); i++) {
      // (a ring longer than the range fills its last stages with the last step again; they are not read)
      const int ks = min(s, nk - 1);
      copy_to(ks, s, i, ks == 0);
    }
  wait_vm((D - 2) * CT + C0);
  lds_barrier();
  if (src.pad > 0) {  // the chunks that do not exist
    const u32x4_t zero = {0u, 0u, 0u, 0u};
    const int xc = src.pad / 8, wc = L::WT == kFp4 ? src.pad / 32 : src.pad / 8;
    for (int e = threadIdx.x; e < L::BM * xc; e += L::THREADS) {
      const int r = e / xc, c = e % xc;
      *(lds_u32x4_t*)(lds + r * L::XROW + 16 * (c ^ L::swx(r))) = zero;
    }
    for (int e = threadIdx.x; e < L::BN * wc; e += L::THREADS) {
      const int r = e / wc, c = e % wc;
      *(lds_u32x4_t*)(lds + L::XB + r * L::WROW + 16 * (c ^ L::sww(r))) = zero;
    }
    lds_barrier();
  }
  if constexpr (NM > 0) {
#pragma unroll
    for (int n = 0; n < NB; n++) read_b(0, 0, n);
#pragma unroll
    for (int m = 0; m < MBV; m++) read_a(0, 0, m);
#pragma unroll
    for (int n = 0; n < NB; n++) convert(0, n);
  }
  int ks = 0;
  for (; ks < nk - D; ks++) step(ks, Int<1>{}, Int<1>{}, Int<1>{});
  if (nk >= D) step(ks++, Int<1>{}, Int<0>{}, Int<1>{});
  for (; ks < nk - 1; ks++) step(ks, Int<0>{}, Int<0>{}, Int<1>{});
  step(ks, Int<0>{}, Int<0>{}, Int<0>{});
  wait_vm(0);
}

// Rows of results from the accumulators to memory: value(mb, nb, r) of column block nb < NBO, to row(tile row) + column
// (null: no such row), columns n0 + 32 NBO wn .. below N, of type YDT.  With vec (rows 16-byte aligned, N a multiple of 16 bytes)
// they leave through LDS, 16 bytes a lane; chunks are permuted so that the two rows of a write (r and r + 4) and
// the rows of a read use distinct banks.  Nontemporal: not read back by this launch.
template <class L, int MBV, int NBO, int YDT, class V, class R>
__device__ __attribute__((always_inline)) inline void store_rows(lds_u8_t* lds, bool vec, int n0, int N, V&& value, R&& row) {
  constexpr int ES = YDT == SMLA_BF16 ? 2 : 4, W = 32 * NBO, CH = W * ES / 16, RPI = 64 / CH;
  constexpr int FIT = L::LDS / (L::NW * 32 * W * ES), REG = L::MB % 2 == 0 && FIT >= 2 ? 2 : 1;
  constexpr int MBP = MBV % REG == 0 ? REG : 1;  // blocks of 32 rows at a time; a wave's region has room for REG
  static_assert(FIT >= 1, "the waves' regions fit the ring's LDS");
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / L::NWN, wn = wave % L::NWN, h = lane >> 5;
  lds_barrier();  // every wave has read its last operands
  if constexpr (MBV > 0) {
    if (vec) {
      lds_u8_t* reg = lds + wave * (REG * 32 * W * ES);
      auto slot = [](int r, int c) { return CH >= 16 ? c ^ ((r << 1) & 8) : c ^ (r & (CH - 1)); };
#pragma unroll
      for (int m0 = 0; m0 < MBV; m0 += MBP) {
#pragma unroll
        for (int mb = 0; mb < MBP; mb++)
#pragma unroll
          for (int nb = 0; nb < NBO; nb++)
#pragma unroll
            for (int r = 0; r < 16; r++) {
              const int rr = 32 * mb + 8 * (r >> 2) + 4 * h + (r & 3), col = (32 * nb + (lane & 31)) * ES;
              lds_u8_t* q = reg + rr * (W * ES) + 16 * slot(rr, col >> 4) + (col & 15);
              const float v = value(m0 + mb, nb, r);
              if constexpr (YDT == SMLA_BF16) *(smla_attn::lds_u16_t*)q = bf16_rne(v);
              else *(smla_attn::lds_f32_t*)q = v;
            }
        const int n = n0 + W * wn + (lane % CH) * (16 / ES);
#pragma unroll
        for (int i = 0; i < MBP * 32 / RPI; i++) {
          const int rr = RPI * i + lane / CH;
          const u32x4_t v = *(lds_u32x4_t*)(reg + rr * (W * ES) + 16 * slot(rr, lane % CH));
          uint8_t* to = row(L::WM * wm + 32 * m0 + rr);
          if (to && n < N) __builtin_nontemporal_store(v, (u32x4_t*)(to + (int64_t)n * ES));
        }
      }
      return;
    }
#pragma unroll
    for (int mb = 0; mb < MBV; mb++)
#pragma unroll
      for (int nb = 0; nb < NBO; nb++) {
        const int n = n0 + W * wn + 32 * nb + (lane & 31);
        if (n >= N) continue;
#pragma unroll
        for (int r = 0; r < 16; r++) {
          uint8_t* to = row(L::WM * wm + 32 * mb + 8 * (r >> 2) + 4 * h + (r & 3));
          if (!to) continue;
          if constexpr (YDT == SMLA_BF16) ((uint16_t*)to)[n] = bf16_rne(value(mb, nb, r));
          else ((float*)to)[n] = value(mb, nb, r);
        }
      }
  }
}

// A workgroup's number in an order in which each XCD takes a contiguous run of `tot` (workgroups are dealt to the
// XCDs in turn); `tot` or more: none.
__device__ inline uint32_t xcd_run(uint32_t tot) {
  const uint32_t per = tot / kXcds, rem = tot % kXcds, x = blockIdx.x % kXcds, i = blockIdx.x / kXcds;
  return i < per + (x < rem) ? x * per + (x < rem ? x : rem) + i : tot;
}

}  // namespace smla_tile
