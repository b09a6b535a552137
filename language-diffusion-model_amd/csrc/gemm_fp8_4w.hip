// 8-bit matrix product for large problems: gemm_mfma4w.hip's four-wave scheme with the scaled 32x32x64 MFMA.
//
// A row of 64 K positions is 64 bytes here as 32 are there, so the ring of five half-tiles of A and B (160 KiB), its
// images, the paired LDS-DMA requests and the one barrier per step are the same; see that file for why.  What differs:
//   * a step is 16 MFMAs of 64 cycles (4 x 4 fragments of 32 x 32 outputs, 256 accumulation registers) instead of 64 of 16:
//     two of the earlier gaps' instructions stand behind each;
//   * a lane's fragment is row lane & 31, chunks h and h + 2 (h = lane >> 5) of its 64 bytes, for both operands alike: which
//     K position a chunk stands for does not matter as long as they agree; the chunks' positions are swizzled for 32 rows;
//   * scales: the MFMA takes one E8M0 byte per row and 32 K positions of either operand.  The bytes of 16 blocks of K
//     (2048 positions) are 16 dwords per lane for A's four row blocks and four for the weights' one block of 128 columns;
//     they are requested before the four steps at the end of the item before, which send nothing else, and moved down by a
//     byte every second step.  Longer K loads the next 16 blocks on the way (one stall in 32 steps);
//   * weight rows are assigned to fragment rows so that a lane holds 32 consecutive columns of a row, and a transposition in the
//     quad leaves 64 consecutive bytes per four lanes in a store: its lane order, not its bytes, decides its time;
//   * all 32 stores go out while the fragments are packed.  Deferring them into the next item's steps, as there, was slower
//     at every share (16384 x 11264 x 2048: 24 deferred 410 us, 16 357, 8 350, none 347): the in-order counter makes the
//     steps' waits for LDS-DMA wait for the stores issued between;
//   * the last tile row or column ends with the matrix and overlaps its neighbour, so M need not be a multiple of 256.
//
// Takes M >= 256, N a multiple of 128 and at least 256, K a multiple of 128 and at least 512; gemm_fp8.hip runs the rest.
// Measured: 8192^3 in 410 us = 2680 TFLOP/s (2683 for the library's product there), 16384 x 11264 x 2048 in 318 us = 2380.  What
// bounds it, by cycle stamps: a step takes 1250 cycles (1330 where K > 2048 loads scales on the way: that load is waited
// for), of which its 16 MFMAs are 1040; with neither reads nor requests it takes the same, so the rest is the addresses,
// scales and loop between the steps.  Packing and storing takes 6000 an item, 11 % at K = 2048.  The clock gives way in turn:
// 2.38 GHz with 16 workgroups, 1.7 to 2.0 with 256, so that 6 % fewer cycles were 2.4 % less time.  Where in a step the
// reads and requests stand made no difference (eight orders within 7 % of the cycles, none faster).
#include <type_traits>

#include "fp8.h"
#include "gemm.h"

namespace {

typedef int i8v __attribute__((ext_vector_type(8)));
typedef int i4v __attribute__((ext_vector_type(4)));
typedef float f4v __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef unsigned u4v_t __attribute__((ext_vector_type(4)));
typedef int i4s_t __attribute__((ext_vector_type(4)));

#define LDS_PTR(p) ((__attribute__((address_space(3))) void *)(p))

constexpr int BM = 256, BN = 256, KH = 64, NSLOT = 5;
constexpr int HT_A = BM * 64, HT_B = BN * 64, HT = HT_A + HT_B;
constexpr int LDS_BYTES = NSLOT * HT;
constexpr int NST = 32;             // stores per wave and item

struct WArgs {
  int64_t M, N, K;
  const uint8_t *A; int64_t lda;
  const uint8_t *sA; int64_t ld_sa;
  const uint8_t *B; int64_t ldb;
  const uint8_t *sB; int64_t ld_sb;
  bf16_t *C; int64_t ldc;
  const float *bias;
  int tiles_m, tiles_n, band_m;
};

// Chunk c of an image row is at position c ^ swz(row): a 128-bit read takes its lanes in groups of 0-3, 12-15, 20-23, 24-27
// and so on, and these positions spread each group's rows over all banks (5.5 cycles a read and CU; 8.0 with the swizzle of
// 16-row fragments).
__device__ __forceinline__ int swz(int row) { return (row >> 2) & 3; }
// Which weight row is which row of a fragment is free; the LDS-DMA's source rows decide it.  Row x of fragment ni is row
// 64 (ni / 2) + 32 ((x / 4) % 2) + 16 (ni % 2) + 4 (x / 8) + x % 4 of the wave's 128: a lane gets register group e = x / 8,
// i = x % 4 for its half of the wave, so over two fragments it ends up with 32 consecutive columns of one row.  Piece i of a
// wave's request (image rows 16 i .. 16 i + 15 of its 64) then has source rows 8 i + this:
__device__ __forceinline__ int src_b(int lane) { return ((lane >> 4) & 1) * 32 + (lane >> 5) * 4 + ((lane >> 2) & 3); }

template <int N>
__device__ __forceinline__ void wait_vm() {
  static_assert(N >= 0 && N <= 63, "vmcnt is a 6-bit counter");
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// accumulator pinned to the accumulation registers; volatile: the MFMAs and the fillers between them stay in order.
// a: weights with their (scalar) scale, b: rows with theirs; the scale's lowest byte counts
__device__ __forceinline__ void mfma_acc(f16v &acc, const i8v &a, const i8v &b, int sa, int sb) {
  asm volatile("v_mfma_scale_f32_32x32x64_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[0,0,0]" : "+a"(acc) : "v"(a), "v"(b), "v"(sa), "v"(sb));
}
__device__ __forceinline__ void mfma_new(f16v &acc, const i8v &a, const i8v &b, int sa, int sb) {
  asm volatile("v_mfma_scale_f32_32x32x64_f8f6f4 %0, %1, %2, 0, %3, %4 op_sel_hi:[0,0,0]" : "=a"(acc) : "v"(a), "v"(b), "v"(sa), "v"(sb));
}

typedef const __attribute__((address_space(4))) WArgs *KArgs;

// First row and column of a tile.  The last tile of a row or column of tiles ends with the matrix: it overlaps its
// neighbour where M or N is no multiple of 256, and both store the same values there.
struct Tile { int m0, n0; };
__device__ __forceinline__ Tile decode_item(int w, int total, KArgs g) {
  const int tiles_m = g->tiles_m, tiles_n = g->tiles_n, band = g->band_m;
  {
    const int q = total >> 3, r = total & 7, x = w & 7;
    w = (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + (w >> 3);
  }
  const int width = band * tiles_n;
  const int grp = w / width;
  const int first = grp * band;
  const int gsz = (tiles_m - first < band) ? tiles_m - first : band;
  const int in = w - grp * width;
  const int m0 = (first + in % gsz) * BM, n0 = in / gsz * BN, ml = (int)g->M - BM, nl = (int)g->N - BN;
  // (the division runs on the vector unit)
  return Tile{__builtin_amdgcn_readfirstlane(m0 < ml ? m0 : ml), __builtin_amdgcn_readfirstlane(n0 < nl ? n0 : nl)};
}

template <int V> using IC = std::integral_constant<int, V>;

struct Scales { int a[4][4], b[4]; };      // [row block][dword], [dword]: 16 blocks of K

// WR: the wave (0..3); wave (wm, wn) = (WR >> 1, WR & 1) owns rows wm * 128.., columns wn * 128.. of the tile
// BIAS = false: no bias loads and additions
template <int WR, bool BIAS>
__device__ __forceinline__ void gemm4w_body(KArgs kp, char *smem) {
  constexpr int wave = WR, wm = WR >> 1, wn = WR & 1;
  // The arguments are read again from the kernel's argument memory wherever an item begins or ends: kept in scalar registers
  // all along they would push the walk's own values out of them.
  auto args = [&]() {
    KArgs p = kp;
    asm volatile("" : "+s"(p));
    return p;
  };
  const int total = kp->tiles_m * kp->tiles_n;
  const int np = (int)(kp->K / KH);
  int w = blockIdx.x;
  if (w >= total) return;
  const unsigned lds_base = (unsigned)(uintptr_t)LDS_PTR(smem);
  const int lane = threadIdx.x & 63;
  // fragment reads: row lane & 31 of a 32-row block; chunk h, and h + 2 (whatever the swizzle, that is the first one's
  // position with bit 1 flipped)
  const unsigned lane_rd = (unsigned)((lane & 31) * 64 + (((lane >> 5) ^ swz(lane & 31)) << 4)) + lds_base;
  const unsigned chunk = (unsigned)(((lane & 3) ^ swz(lane >> 2)) << 4);
  const unsigned laneA = (unsigned)(lane >> 2) * (unsigned)kp->lda + chunk;
  const unsigned laneB = (unsigned)src_b(lane) * (unsigned)kp->ldb + chunk;
  const unsigned lane_st = (unsigned)(((lane >> 2) & 7) * 4 * (int)kp->ldc * 2 + (lane & 3) * 16 + (lane >> 5) * 64);
  // piece i of a wave's four (16 rows each; B's are 8 rows apart, see src_b); the immediate i * 1024 also advances the LDS address, so base_i is 1024 i lower
  const char *bA[4], *bB[4];
  auto dma = [&](auto I, bool opB, unsigned voff) {
    constexpr int i = decltype(I)::value;
    const char *base = opB ? bB[i] : bA[i];
    asm volatile("global_load_lds_dwordx4 %0, %1 offset:%2" ::"v"(voff), "s"(base), "n"(i * 1024) : "memory");
  };
  auto set_m0 = [&](unsigned v) { asm volatile("s_mov_b32 m0, %0\n\ts_nop 0" ::"s"(v) : "memory"); };
  auto m0_of = [&](int h, bool opB) { return lds_base + (h % NSLOT) * HT + (opB ? HT_A : 0) + wave * 4096; };
  auto prologue = [&](Tile t) {
    const KArgs g = args();
    const int64_t pieceA = (int64_t)16 * g->lda - 1024, pieceB = (int64_t)8 * g->ldb - 1024;
    const char *tA = (const char *)(g->A + ((int64_t)t.m0 + wave * 64) * g->lda);
    const char *tB = (const char *)(g->B + ((int64_t)t.n0 + wave * 64) * g->ldb);
#pragma unroll
    for (int i = 0; i < 4; ++i) { bA[i] = tA + i * pieceA; bB[i] = tB + i * pieceB; }
    auto pair = [&](int h) {
      const unsigned va = laneA + h * 64, vb = laneB + h * 64;
      const unsigned a0 = m0_of(h, false), a1 = m0_of(h + 1, false), b0 = m0_of(h, true), b1 = m0_of(h + 1, true);
      set_m0(a0); dma(IC<0>{}, false, va); set_m0(a1); dma(IC<0>{}, false, va + 64);
      set_m0(a0); dma(IC<1>{}, false, va); set_m0(a1); dma(IC<1>{}, false, va + 64);
      set_m0(a0); dma(IC<2>{}, false, va); set_m0(a1); dma(IC<2>{}, false, va + 64);
      set_m0(a0); dma(IC<3>{}, false, va); set_m0(a1); dma(IC<3>{}, false, va + 64);
      set_m0(b0); dma(IC<0>{}, true, vb); set_m0(b1); dma(IC<0>{}, true, vb + 64);
      set_m0(b0); dma(IC<1>{}, true, vb); set_m0(b1); dma(IC<1>{}, true, vb + 64);
      set_m0(b0); dma(IC<2>{}, true, vb); set_m0(b1); dma(IC<2>{}, true, vb + 64);
      set_m0(b0); dma(IC<3>{}, true, vb); set_m0(b1); dma(IC<3>{}, true, vb + 64);
    };
    pair(0);
    pair(2);
  };
  // Blocks c0 .. c0 + 15 of K.  Dwords at any byte alignment; the last one of a row is read four bytes before the row's end
  // (never behind it) and shifted down: nb >= 4, and c0 > 0 has 16 bytes in front.
  auto load_scales = [&](Scales &s, Tile t, int c0) {
    const KArgs g = args();
    const int rem = (np >> 1) - c0;
    int row = lane & 31;
    asm volatile("" : "+v"(row));      // (computed here: hoisted out of the loop, the addresses cost registers all along)
    const uint8_t *pa = g->sA + ((int64_t)t.m0 + wm * 128 + row) * g->ld_sa + c0;
    const uint8_t *pb = g->sB + (int64_t)(t.n0 / FP8_BLOCK + wn) * g->ld_sb + c0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int off = 4 * j < rem - 4 ? 4 * j : rem - 4;
      const int o = off < 0 ? (c0 ? off : 0) : off;      // (dwords that do not exist read the row's first bytes)
      int v;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        __builtin_memcpy(&v, pa + (int64_t)32 * i * g->ld_sa + o, 4);
        s.a[i][j] = v;
      }
      __builtin_memcpy(&v, pb + o, 4);
      s.b[j] = v;
    }
  };
  auto settle_scales = [&](Scales &s, int c0) {
    const int rem = (np >> 1) - c0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int sh = 4 * j < rem - 4 ? 0 : (4 * j - (rem - 4)) * 8;     // (32 and more: a dword that is not used)
#pragma unroll
      for (int i = 0; i < 4; ++i) s.a[i][j] = (int)((unsigned)s.a[i][j] >> (sh & 31));
      s.b[j] = (int)((unsigned)s.b[j] >> (sh & 31));
    }
  };
  auto frag = [&](unsigned va, int off) {
    return *reinterpret_cast<const __attribute__((address_space(3))) i4v *>((uintptr_t)(va + off));
  };
  auto store_q = [&](const u4v_t &q, const i4s_t &srd, unsigned soff, auto T) {
    constexpr int t = decltype(T)::value;
    const unsigned vo = lane_st;
    asm volatile("buffer_store_dwordx4 %0, %1, %2, %3 offen offset:%4\n\ts_nop 0" ::"v"(q), "v"(vo), "s"(srd), "s"(soff), "n"(t * 128) : "memory");
  };

  Tile tid = decode_item(w, total, args());
  Scales sc;
  load_scales(sc, tid, 0);
  settle_scales(sc, 0);
  prologue(tid);
  bool first_item = true;

  while (true) {
    f16v acc[4][4];
    i4v fal[2][4], fah[2][4], fbl[2][4], fbh[2][4];

    // half-tiles 0, 1 landed.  Issue order of this wave's vector-memory instructions: prologue (32) | stores
    // of the packing phase (not before the first item) | step 0 ...
    const bool stores_behind = !first_item;
    if (stores_behind) wait_vm<16 + NST>(); else wait_vm<16>();
    first_item = false;
    __builtin_amdgcn_s_waitcnt(0xC07F);   // lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    {
      const unsigned lo = lane_rd, hi = lane_rd ^ 32;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        fal[0][i] = frag(lo, wm * 8192 + i * 2048);
        fah[0][i] = frag(hi, wm * 8192 + i * 2048);
        fbl[0][i] = frag(lo, HT_A + wn * 8192 + i * 2048);
        fbh[0][i] = frag(hi, HT_A + wn * 8192 + i * 2048);
      }
    }

    // One 64-deep step: MFMAs on the fragments of half-tile p (set cur) with, behind them, the reads of half-tile p+1 (set
    // nxt) and this step's LDS-DMA.
    //   PAR = p & 1; FIRST: step 0 or 1 (step 0: C = 0); ISSUE: the step sends LDS-DMA; LAST: the item's last step, which
    //   reads no half-tile ahead and requests this lane's columns of the bias into the registers of that
    [[maybe_unused]] f4v bv[16];
    auto step = [&](auto PAR, auto FIRST, auto ISSUE, auto LAST, int p) {
      constexpr int cur = decltype(PAR)::value, nxt = cur ^ 1;
      constexpr bool first = decltype(FIRST)::value;
      constexpr bool do_issue = decltype(ISSUE)::value, last = decltype(LAST)::value;
      // An odd step needs the pair (p+1, p+2) complete.  Its last request went out in step p-2 (or before the item); younger
      // are the eight requests of step p-1, and for step 1 the stores of the item before.
      if constexpr (cur == 1) {
        if constexpr (!do_issue) {
          wait_vm<0>();
        } else if constexpr (first) {
          if (stores_behind) wait_vm<8 + NST>(); else wait_vm<8>();
        } else {
          wait_vm<8>();
        }
      }
      if constexpr (cur == 0 && !first) {
        // the next block of K: its byte moves to the bottom
        if ((p & 31) == 0) {
          load_scales(sc, tid, p >> 1);
          settle_scales(sc, p >> 1);
        } else if ((p & 7) == 0) {
          asm volatile("");      // (a branch: as selections this is 30 vector instructions in every second step)
#pragma unroll
          for (int j = 0; j < 3; ++j) {
            sc.b[j] = sc.b[j + 1];
#pragma unroll
            for (int i = 0; i < 4; ++i) sc.a[i][j] = sc.a[i][j + 1];
          }
        } else {
          sc.b[0] = (int)((unsigned)sc.b[0] >> 8);
#pragma unroll
          for (int i = 0; i < 4; ++i) sc.a[i][0] = (int)((unsigned)sc.a[i][0] >> 8);
        }
      }
      const int hpair = cur == 0 ? p + 4 : p + 3;
      unsigned voff = (cur == 1 ? laneB : laneA) + hpair * 64;
      unsigned voff2 = voff + 64;
      unsigned mA = m0_of(hpair, cur == 1), mB = m0_of(hpair + 1, cur == 1);
      unsigned lo = lane_rd + ((p + 1) % NSLOT) * HT, hi = lo ^ 32;      // (slots are multiples of 32 KiB: bit 5 is the lane's)
      asm volatile("" : "+v"(lo), "+v"(hi), "+v"(voff), "+v"(voff2), "+s"(mA), "+s"(mB));
      asm volatile("" : "+v"(sc.a[0][0]), "+v"(sc.a[1][0]), "+v"(sc.a[2][0]), "+v"(sc.a[3][0]), "+v"(sc.b[0]));
      __builtin_amdgcn_s_waitcnt(0xC07F);   // lgkmcnt(0): this wave's reads of half-tile p are complete
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_barrier();
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (last && BIAS) {
        const float *bb = args()->bias + tid.n0 + wn * 128 + (lane >> 5) * 32;
#pragma unroll
        for (int i = 0; i < 16; ++i) bv[i] = *reinterpret_cast<const f4v *>(bb + (i / 8) * 64 + (i % 8) * 4);
        __builtin_amdgcn_sched_barrier(0);
      }
      // Gap s (two behind each MFMA), period of eight gaps, gq = s % 8, j = s / 8: LDS-DMA of piece j in gaps 2 WR and
      // 2 WR + 1, fragment reads in the first four of the others
      auto filler = [&](auto S) {
        constexpr int s_ = decltype(S)::value, gq = s_ % 8, j = s_ / 8;
        if constexpr (gq == 2 * WR || gq == 2 * WR + 1) {
          if constexpr (do_issue) {
            set_m0(gq == 2 * WR ? mA : mB);
            dma(IC<j>{}, cur == 1, gq == 2 * WR ? voff : voff2);
          }
        } else if constexpr (!last) {
          constexpr int rank = gq - (gq > 2 * WR ? 2 : 0);
          if constexpr (rank < 4) {
            if constexpr (rank == 0) fal[nxt][j] = frag(lo, wm * 8192 + j * 2048);
            else if constexpr (rank == 1) fah[nxt][j] = frag(hi, wm * 8192 + j * 2048);
            else if constexpr (rank == 2) fbl[nxt][j] = frag(lo, HT_A + wn * 8192 + j * 2048);
            else fbh[nxt][j] = frag(hi, HT_A + wn * 8192 + j * 2048);
          }
        }
      };
      auto run = [&](auto self, auto K) {
        constexpr int k = decltype(K)::value;
        if constexpr (k < 16) {
          constexpr int gi = k / 4, ni = k % 4;
          const i8v a = __builtin_shufflevector(fbl[cur][ni], fbh[cur][ni], 0, 1, 2, 3, 4, 5, 6, 7);
          const i8v b = __builtin_shufflevector(fal[cur][gi], fah[cur][gi], 0, 1, 2, 3, 4, 5, 6, 7);
          if constexpr (first && cur == 0) mfma_new(acc[ni][gi], a, b, sc.b[0], sc.a[gi][0]);
          else mfma_acc(acc[ni][gi], a, b, sc.b[0], sc.a[gi][0]);
          __builtin_amdgcn_sched_barrier(0);
          filler(IC<2 * k>{});
          __builtin_amdgcn_sched_barrier(0);
          filler(IC<2 * k + 1>{});
          __builtin_amdgcn_sched_barrier(0);
          self(self, IC<k + 1>{});
        }
      };
      run(run, IC<0>{});
    };
    typedef std::true_type T_;
    typedef std::false_type F_;
    step(IC<0>{}, T_{}, T_{}, F_{}, 0);
    step(IC<1>{}, T_{}, T_{}, F_{}, 1);
    int p = 2;
    for (; p < np - 4; p += 2) {
      step(IC<0>{}, F_{}, T_{}, F_{}, p);
      step(IC<1>{}, F_{}, T_{}, F_{}, p + 1);
    }
    // the last four steps send no LDS-DMA: the next item's scales are requested in front of them (without a next item: this
    // one's again, unused)
    w += gridDim.x;
    const bool more = w < total;
    const Tile next = more ? decode_item(w, total, args()) : tid;
    Scales sn;
    load_scales(sn, next, 0);
    step(IC<0>{}, F_{}, F_{}, F_{}, p);
    step(IC<1>{}, F_{}, F_{}, F_{}, p + 1);
    step(IC<0>{}, F_{}, F_{}, F_{}, p + 2);
    step(IC<1>{}, F_{}, F_{}, T_{}, p + 3);
    // (the asm MFMAs' results: wait states the compiler does not count)
    asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
    settle_scales(sn, 0);
    sc = sn;
    // (waited for here: behind the next item's prologue the in-order counter would wait for that as well)
    if constexpr (BIAS) {
#pragma unroll
      for (int i = 0; i < 16; ++i) asm volatile("" : "+v"(bv[i]));
    }

    const Tile here = tid;
    tid = next;
    if (more) prologue(tid);
    // Pack: fragments (gi, 2 half) and (gi, 2 half + 1) = rows gi * 32 .., a lane's 32 columns from 64 half + 32 h: four pieces of 8
    // columns.  Transposing them in the quad leaves 64 consecutive bytes per four lanes, 8 rows x 128 bytes per store.
    {
      const KArgs g = args();
      const char *cb = (const char *)(g->C + (int64_t)(here.m0 + wm * 128) * g->ldc + here.n0 + wn * 128);
      i4s_t srd;
      srd[0] = (int)(uintptr_t)cb;
      srd[1] = (int)(((uintptr_t)cb >> 32) & 0xffff);
      srd[2] = -1;
      srd[3] = 0x00020000;
      auto rd4 = [&](auto E, const f16v &x) {
        constexpr int e = decltype(E)::value * 4;
        f4v r;
        asm volatile("v_accvgpr_read_b32 %0, %4\n\tv_accvgpr_read_b32 %1, %5\n\tv_accvgpr_read_b32 %2, %6\n\tv_accvgpr_read_b32 %3, %7"
                     : "=v"(r[0]), "=v"(r[1]), "=v"(r[2]), "=v"(r[3]) : "a"(x[e]), "a"(x[e + 1]), "a"(x[e + 2]), "a"(x[e + 3]));
        return r;
      };
      const unsigned ldc2 = (unsigned)(g->ldc * 2);     // bytes per row of C
      auto packq = [&](auto self, auto C) {
        constexpr int c = decltype(C)::value;
        if constexpr (c < 8) {
          constexpr int gi = c / 2, half = c % 2;
          unsigned q[4][4];      // [dword][piece]
          auto grp = [&](auto P, auto E) {
            constexpr int piece = decltype(P)::value, ni = half * 2 + piece / 2, e = (piece % 2) * 2 + decltype(E)::value;
            f4v v = rd4(IC<e>{}, acc[ni][gi]);
            if constexpr (BIAS) v += bv[ni * 4 + e];
            q[decltype(E)::value * 2][piece] = pack_bf16x2(v[0], v[1]);
            q[decltype(E)::value * 2 + 1][piece] = pack_bf16x2(v[2], v[3]);
          };
          grp(IC<0>{}, IC<0>{}); grp(IC<0>{}, IC<1>{}); grp(IC<1>{}, IC<0>{}); grp(IC<1>{}, IC<1>{});
          grp(IC<2>{}, IC<0>{}); grp(IC<2>{}, IC<1>{}); grp(IC<3>{}, IC<0>{}); grp(IC<3>{}, IC<1>{});
          quad_transpose4(q);
#pragma unroll
          for (int t = 0; t < 4; ++t) store_q(u4v_t{q[0][t], q[1][t], q[2][t], q[3][t]}, srd, (unsigned)(gi * 32 + t) * ldc2, IC<half>{});
          __builtin_amdgcn_sched_barrier(0);
          self(self, IC<c + 1>{});
        }
      };
      packq(packq, IC<0>{});
    }
    if (!more) break;
  }
}

template <bool BIAS>
__global__ __launch_bounds__(256, 1) void gemm_fp8_4w_k(WArgs) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const KArgs kp = (KArgs)__builtin_amdgcn_kernarg_segment_ptr();      // the one argument is at its start
  // one copy of the code per wave: the copies differ in which gap of a step holds what
  if (wave == 0) gemm4w_body<0, BIAS>(kp, smem);
  else if (wave == 1) gemm4w_body<1, BIAS>(kp, smem);
  else if (wave == 2) gemm4w_body<2, BIAS>(kp, smem);
  else gemm4w_body<3, BIAS>(kp, smem);
}

}  // namespace

int ldm_gemm_fp8_4w(int64_t M, int64_t N, int64_t K, const uint8_t *A, int64_t lda, const uint8_t *sA, int64_t ld_sa,
                    const uint8_t *B, int64_t ldb, const uint8_t *sB, int64_t ld_sb, void *C, int64_t ldc,
                    const float *bias, hipStream_t s) {
  if (M < 256 || N < 256 || N % FP8_BLOCK) return LDM_E_SHAPE;
  if (K % FP8_BLOCK || K < 4 * FP8_BLOCK) return LDM_E_SHAPE;      // (four bytes of scales per row, six steps)
  if (lda % 16 || ldb % 16 || ldc % 8 || !aligned_to(A, 16) || !aligned_to(B, 16) || !aligned_to(C, 16) ||
      (bias && !aligned_to(bias, 16)))
    return LDM_E_ALIGN;
  // Lane offsets are unsigned 32-bit: up to 15 rows of A and 39 of B (src_b) plus K <= ldb, 40 x 2^26 < 2^32; 128 rows of C
  // (2 ldc bytes each), 2^31
  if (lda >= (1 << 26) || ldb >= (1 << 26) || ldc >= (1 << 23)) return LDM_E_SHAPE;
  const int64_t tm = ceil_div(M, 256), tn = ceil_div(N, 256);
  if (M > 0x7fffff00 || N > 0x7fffff00 || tm * tn > 0x3fffffff) return LDM_E_SHAPE;
  WArgs g;
  g.M = M; g.N = N; g.K = K;
  g.A = A; g.lda = lda; g.sA = sA; g.ld_sa = ld_sa;
  g.B = B; g.ldb = ldb; g.sB = sB; g.ld_sb = ld_sb;
  g.C = (bf16_t *)C; g.ldc = ldc; g.bias = bias;
  g.tiles_m = (int)tm; g.tiles_n = (int)tn;
  int b = 8;
  while (b > 2 && (int64_t)b * 256 * K > (int64_t)8 << 20) b >>= 1;
  g.band_m = b;
  static std::atomic<uint64_t> attr_done{0};
  uint64_t dev_bit;
  if (ldm_attr_pending(attr_done, &dev_bit)) {
    (void)hipFuncSetAttribute((const void *)gemm_fp8_4w_k<false>, hipFuncAttributeMaxDynamicSharedMemorySize, LDS_BYTES);
    (void)hipFuncSetAttribute((const void *)gemm_fp8_4w_k<true>, hipFuncAttributeMaxDynamicSharedMemorySize, LDS_BYTES);
    attr_done.fetch_or(dev_bit, std::memory_order_release);
  }
  const int64_t items = tm * tn, cus = 256;
  const dim3 grid((unsigned)(items < cus ? items : cus)), wg(256);
  if (bias) hipLaunchKernelGGL(gemm_fp8_4w_k<true>, grid, wg, LDS_BYTES, s, g);
  else hipLaunchKernelGGL(gemm_fp8_4w_k<false>, grid, wg, LDS_BYTES, s, g);
  LDM_CHECK_LAUNCH();
  return LDM_OK;
}
