// 8-bit matrix product of the inference projections on the scaled MFMA of gfx950:
//   C[m, n] = sum_kb 2^(ea[m, kb] + eb[n / 128, kb]) * sum_{k in block kb} A[m, k] * B[n, k]  (+ bias[n])
// A [M, K] e4m3 rows with one E8M0 scale per 128 columns, B [N, K] e4m3 weights with one per 128 x 128 block, fp32
// accumulation, bf16 or fp32 output.
//
// bf16 output: v_mfma_scale_f32_16x16x128_f8f6f4 takes an E8M0 scale per row and 32 values of either operand: power-of-two
// scales cost no vector instruction, where a general fp32 scale would need one multiply-add per accumulator and block
// beside the matrix pipe (about half its time again).  Precision, measured: of the eight products of a lane's consecutive
// K positions each is truncated at 2^-13 of the leading bit of the largest; the groups of eight are added in fp32.  Random
// operands lose 1.5e-5 of the result (2-norm), well below the bf16 rounding of the output (1.7e-3), but far above fp32's.
//
// fp32 output: the unscaled 8-bit MFMA truncates likewise, the bf16 one does not (one product of 32 positions of e4m3 values
// is within 2^-22 of the sum of their magnitudes, 5e-8 in the 2-norm).  e4m3 values are bf16 values, so the fragments are
// widened in registers and four 16x16x32 bf16 MFMAs form a block's sum, which ldexp scales into the accumulator: half the
// matrix rate, and two vector instructions per accumulator and block.
#include <type_traits>

#include "fp8.h"
#include "gemm.h"

namespace {

typedef int i8v __attribute__((ext_vector_type(8)));
typedef int i4v __attribute__((ext_vector_type(4)));
typedef float f4v __attribute__((ext_vector_type(4)));

struct GArgs {
  int64_t M, N, K;
  const uint8_t *A; int64_t lda;
  const uint8_t *sA; int64_t ld_sa;
  const uint8_t *B; int64_t ldb;
  const uint8_t *sB; int64_t ld_sb;
  const float *bias;
  void *C; int64_t ldc;
};

__device__ __forceinline__ f4v mfma_scaled(const i8v &a, const i8v &b, const f4v &c, int sa, int sb) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, sa, 0, sb);
}

// 16 bytes of a row at column k: bytes at and beyond K are zeros (a row is readable to the next multiple of 16)
__device__ __forceinline__ i4v load16_tail(const uint8_t *row, int64_t k, int64_t K) {
  i4v v = {0, 0, 0, 0};
  if (k >= K) return v;
  v = *reinterpret_cast<const i4v *>(row + k);
  const int left = (int)(K - k);
  if (left < 16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int b = left - 4 * i;
      v[i] = b >= 4 ? v[i] : b <= 0 ? 0 : (int)((unsigned)v[i] & (0xffffffffu >> (32 - 8 * b)));
    }
  }
  return v;
}
__device__ __forceinline__ i8v join(const i4v &a, const i4v &b) {
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// fp32 output: a fragment's 32 values as four bf16 operands (positions 8 s .. 8 s + 7 of the lane's 32 in operand s, of either
// side alike)
typedef __bf16 b8v __attribute__((ext_vector_type(8)));
typedef __bf16 b2v __attribute__((ext_vector_type(2)));
struct Wide { b8v s[4]; };
__device__ __forceinline__ Wide widen(const i8v &x) {
  Wide w;
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    i4v d;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const b2v lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)x[2 * s + h], 1.0f, false);
      const b2v hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)x[2 * s + h], 1.0f, true);
      d[2 * h] = __builtin_bit_cast(int, lo);
      d[2 * h + 1] = __builtin_bit_cast(int, hi);
    }
    w.s[s] = __builtin_bit_cast(b8v, d);
  }
  return w;
}
// acc[j] += 2^(ea + eb) * (b[j] . a), from the scales' codes (255 is NaN).  ldexp, for the power itself may lie outside fp32
// where the result does not.
template <int TN>
__device__ __forceinline__ void add_block(f4v (&acc)[TN], const Wide (&b)[TN], const Wide &a, int ea, int eb) {
  const float c0 = ea == 255 || eb == 255 ? __builtin_nanf("") : 0.f;
  const int e = ea + eb - 254;
  f4v p[TN];
#pragma unroll
  for (int j = 0; j < TN; ++j) p[j] = f4v{c0, c0, c0, c0};
#pragma unroll
  for (int s = 0; s < 4; ++s)
#pragma unroll
    for (int j = 0; j < TN; ++j) p[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[j].s[s], a.s[s], p[j], 0, 0, 0);
#pragma unroll
  for (int j = 0; j < TN; ++j)
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[j][k] += ldexpf(p[j][k], e);
}
// one 16 x 16 block of outputs, either way
template <typename OT>
__device__ __forceinline__ void add_one(f4v &acc, const i8v &b, const i8v &a, int ea, int eb) {
  if constexpr (std::is_same_v<OT, float>) {
    f4v t[1] = {acc};
    const Wide w[1] = {widen(b)};
    add_block(t, w, widen(a), ea, eb);
    acc = t[0];
  } else {
    acc = mfma_scaled(b, a, acc, eb, ea);
  }
}

// four consecutive columns of a row of C
template <typename OT>
__device__ __forceinline__ void store4(const GArgs &g, int64_t m, int64_t n, f4v v, bool vec) {
  if (m >= g.M || n >= g.N) return;
  OT *c = (OT *)g.C + m * g.ldc + n;
  if (n + 4 <= g.N) {
    if (g.bias) {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] += g.bias[n + j];
    }
    if (vec) {
      st4(c, f4{{v[0], v[1], v[2], v[3]}});
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) Elt<OT>::st(c + j, v[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (n + j < g.N) Elt<OT>::st(c + j, v[j] + (g.bias ? g.bias[n + j] : 0.f));
  }
}

// Few rows: the weights are the traffic.  A workgroup owns 16 columns and 16 * MT rows, its four waves split the
// blocks of K and add up through LDS; fragments come straight from memory (a 16 x 128-byte fragment is 16 whole lines).
// The weights are the FIRST operand, so a lane ends up with four consecutive columns of one row.
template <int MT, typename OT>
__global__ __launch_bounds__(256) void gemm_fp8_rows_k(GArgs g, bool vec) {
  __shared__ f4v red[4][MT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 15, q = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * 16, m0 = (int64_t)blockIdx.y * (16 * MT);
  const int64_t n = n0 + r < g.N ? n0 + r : g.N - 1;
  const uint8_t *b = g.B + n * g.ldb;
  const uint8_t *sb = g.sB + (n0 / FP8_BLOCK) * g.ld_sb;
  const uint8_t *a[MT], *sa[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int64_t m = m0 + i * 16 + r < g.M ? m0 + i * 16 + r : g.M - 1;
    a[i] = g.A + m * g.lda;
    sa[i] = g.sA + m * g.ld_sa;
  }
  f4v acc[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) acc[i] = f4v{0.f, 0.f, 0.f, 0.f};
  const int full = (int)(g.K / FP8_BLOCK), nkb = (int)((g.K + FP8_BLOCK - 1) / FP8_BLOCK);
  int kb = wave;
  for (; kb < full; kb += 4) {
    const int64_t k = (int64_t)kb * FP8_BLOCK + q * 32;
    const i8v fb = join(*reinterpret_cast<const i4v *>(b + k), *reinterpret_cast<const i4v *>(b + k + 16));
    const int eb = sb[kb];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const i8v fa = join(*reinterpret_cast<const i4v *>(a[i] + k), *reinterpret_cast<const i4v *>(a[i] + k + 16));
      add_one<OT>(acc[i], fb, fa, sa[i][kb], eb);
    }
  }
  if (kb < nkb) {
    const int64_t k = (int64_t)kb * FP8_BLOCK + q * 32;
    const i8v fb = join(load16_tail(b, k, g.K), load16_tail(b, k + 16, g.K));
    const int eb = sb[kb];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const i8v fa = join(load16_tail(a[i], k, g.K), load16_tail(a[i], k + 16, g.K));
      add_one<OT>(acc[i], fb, fa, sa[i][kb], eb);
    }
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) red[wave][i][lane] = acc[i];
  __syncthreads();
  for (int t = threadIdx.x; t < MT * 64; t += 256) {
    const int i = t >> 6, l = t & 63;
    const f4v v = (red[0][i][l] + red[1][i][l]) + (red[2][i][l] + red[3][i][l]);
    store4<OT>(g, m0 + i * 16 + (l & 15), n0 + (l >> 4) * 4, v, vec);
  }
}

// Tiles through LDS: BM x 128 outputs per workgroup of 2 x 2 waves, each 16 * TM rows by 64 columns.  One block of K (128
// bytes of every row) per step, two steps in LDS: the next one is requested as soon as every wave has finished the one before
// (one barrier per step), so it has a whole step to arrive.  Two workgroups of 128 x 128 share a CU (64 KiB of tiles plus
// the scales each; three of 64 x 128): one's stores and waits run under the other's products.
//
// LDS image of an operand: [rows][128 bytes], the 16-byte chunk c of row r at position c ^ (bit 1 of r | 4 * bit 3 of r), of a
// weights' row c ^ (bit 1 of r | 4 * bit 5 of r).  A 128-bit read takes its lanes in groups of 0-3, 12-15, 20-23, 24-27 and so
// on; with these positions each group covers all banks (5.5 cycles a read and CU; 8.0 with c ^ (r & 7)).  LDS-DMA
// writes lane-linearly, so the swizzle is on its source.
//
// Which weight row is which row of a fragment is free: lane r of fragment j reads row 16 * (r / 4) + 4 * j + r % 4 of the
// wave's 64, so that a lane ends up with 16 consecutive columns of one row over the four fragments.
// Scales of 64 steps are kept as [step][row], a lane's TM rows side by side (one read per step).
constexpr int SCH = 64;      // steps whose scales are in LDS at a time

#define LDM_LDS_PTR(p) ((__attribute__((address_space(3))) void *)(p))

// 16 bytes per lane from base + off to LDS at lds + lane * 16 (the write of m0 needs one wait state before its use)
__device__ __forceinline__ void lds_dma16(unsigned lds, unsigned off, const uint8_t *base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base) : "memory");
}

template <int TM, typename OT>
__global__ __launch_bounds__(256, 2) void gemm_fp8_tile_k(GArgs g, int tiles_m, int tiles_n, int band, bool vec) {
  constexpr int BM = 32 * TM, BN = FP8_BLOCK, TN = 4;
  constexpr int STAGE = (BM + BN) * FP8_BLOCK;
  constexpr int DA = BM / 32, DB = BN / 32;            // LDS-DMA requests (8 rows each) per wave and step
  extern __shared__ __attribute__((aligned(16))) char smem[];
  uint8_t *sca = (uint8_t *)smem + 2 * STAGE;          // [SCH][BM]
  uint8_t *scb = sca + SCH * BM;                       // [SCH]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave >> 1, wn = wave & 1, r = lane & 15, q = lane >> 4;
  // consecutive workgroups go to different XCDs: give each XCD a contiguous run of tiles, walked in bands of `band` row
  // tiles, so that the workgroups that share an L2 share operand panels
  int tm, tn;
  {
    const int total = tiles_m * tiles_n;
    int w = blockIdx.x;
    const int per = total >> 3, rem = total & 7, x = w & 7;
    w = (x < rem ? x * (per + 1) : rem * (per + 1) + (x - rem) * per) + (w >> 3);
    const int width = band * tiles_n, grp = w / width, first = grp * band;
    const int gsz = tiles_m - first < band ? tiles_m - first : band;
    const int in = w - grp * width;
    tm = first + in % gsz;
    tn = in / gsz;
  }
  const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
  const int mrows = (int)(g.M - m0 < BM ? g.M - m0 : BM), nrows = (int)(g.N - n0 < BN ? g.N - n0 : BN);
  const int full = (int)(g.K / FP8_BLOCK), krem = (int)(g.K % FP8_BLOCK), nkb = full + (krem ? 1 : 0);
  const uint8_t *baseA = g.A + m0 * g.lda, *baseB = g.B + n0 * g.ldb;
  // source offsets: request j of this wave holds rows (wave * D + j) * 8 + lane / 8; rows behind the last one repeat it
  unsigned offA[DA], offB[DB];
  static_assert(DA % 2 == 0 && DB == 4, "bit 3 of a row is the request's lowest bit, bit 5 of a weights' row the wave's");
  auto chunkA = [&](int j) { return (lane & 7) ^ ((lane >> 4) & 1) ^ ((j & 1) << 2); };
  const int chunkB = (lane & 7) ^ ((lane >> 4) & 1) ^ ((wave & 1) << 2);
#pragma unroll
  for (int j = 0; j < DA; ++j) {
    const int row = (wave * DA + j) * 8 + (lane >> 3);
    offA[j] = (unsigned)((row < mrows ? row : mrows - 1) * (int)g.lda + chunkA(j) * 16);
  }
#pragma unroll
  for (int j = 0; j < DB; ++j) {
    const int row = (wave * DB + j) * 8 + (lane >> 3);
    offB[j] = (unsigned)((row < nrows ? row : nrows - 1) * (int)g.ldb + chunkB * 16);
  }
  const unsigned lds0 = (unsigned)(uintptr_t)LDM_LDS_PTR(smem);
  auto request = [&](int kb) {
    if (kb == full) {      // the partial block: chunks behind column K are not read (chunk 0 again; masked after the read)
      auto back = [&](int chunk) { return chunk * 16 >= krem ? (unsigned)(chunk * 16) : 0u; };
#pragma unroll
      for (int j = 0; j < DA; ++j) offA[j] -= back(chunkA(j));
#pragma unroll
      for (int j = 0; j < DB; ++j) offB[j] -= back(chunkB);
    }
    const uint8_t *a = baseA + (int64_t)kb * FP8_BLOCK, *b = baseB + (int64_t)kb * FP8_BLOCK;
    const unsigned la = lds0 + (kb & 1) * STAGE + wave * (DA * 1024), lb = lds0 + (kb & 1) * STAGE + BM * FP8_BLOCK + wave * (DB * 1024);
#pragma unroll
    for (int j = 0; j < DA; ++j) lds_dma16(la + j * 1024, offA[j], a);
#pragma unroll
    for (int j = 0; j < DB; ++j) lds_dma16(lb + j * 1024, offB[j], b);
  };
  auto load_scales = [&](int kb0) {
    const int n = nkb - kb0 < SCH ? nkb - kb0 : SCH;
    constexpr int PER = 256 / BM;       // threads per row
    const int row = threadIdx.x / PER;
    const uint8_t *s = g.sA + (m0 + (row < mrows ? row : mrows - 1)) * g.ld_sa + kb0;
    // row = (wave row, i, r): position wave row * 16 TM + r * TM + i
    const int pos = (row / (16 * TM)) * (16 * TM) + (row & 15) * TM + ((row / 16) & (TM - 1));
    for (int k = threadIdx.x % PER; k < n; k += PER) sca[k * BM + pos] = s[k];
    if (threadIdx.x < n) scb[threadIdx.x] = g.sB[tn * g.ld_sb + kb0 + threadIdx.x];
  };
  f4v acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f4v{0.f, 0.f, 0.f, 0.f};
  request(0);
  load_scales(0);
  // fragment of 16 rows: chunks 2q and 2q + 1 (the first one's position with bit 0 flipped) of a row's 128 bytes
  const int pos = ((2 * q) ^ ((r >> 1) & 1) ^ ((r >> 3) << 2)) << 4;
  const int rdA = r * FP8_BLOCK + pos, rdB = ((r >> 2) * 16 + (r & 3)) * FP8_BLOCK + pos;
  auto step = [&](int kb, auto TAIL) {
    constexpr bool tail = decltype(TAIL)::value;
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (kb && (kb % SCH) == 0) {
      load_scales(kb);
      __syncthreads();
    }
    if (kb + 1 < nkb) request(kb + 1);
    const char *sa = smem + (kb & 1) * STAGE + wm * (16 * TM * FP8_BLOCK);
    const char *sb = smem + (kb & 1) * STAGE + BM * FP8_BLOCK + wn * (16 * TN * FP8_BLOCK);
    auto frag = [&](const char *p, int rd) {
      i4v lo = *reinterpret_cast<const i4v *>(p + rd), hi = *reinterpret_cast<const i4v *>(p + (rd ^ 16));
      if constexpr (tail) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int bl = krem - q * 32 - 4 * i, bh = bl - 16;
          lo[i] = bl >= 4 ? lo[i] : bl <= 0 ? 0 : (int)((unsigned)lo[i] & (0xffffffffu >> (32 - 8 * bl)));
          hi[i] = bh >= 4 ? hi[i] : bh <= 0 ? 0 : (int)((unsigned)hi[i] & (0xffffffffu >> (32 - 8 * bh)));
        }
      }
      return join(lo, hi);
    };
    const int eb = scb[kb % SCH];
    int ea[(TM + 3) / 4];
#pragma unroll
    for (int i = 0; i < (TM + 3) / 4; ++i) {
      const uint8_t *p = sca + (kb % SCH) * BM + wm * (16 * TM) + r * TM + 4 * i;
      ea[i] = TM >= 4 ? *reinterpret_cast<const int *>(p) : *reinterpret_cast<const unsigned short *>(p);
    }
    i8v fb[TN];
#pragma unroll
    for (int j = 0; j < TN; ++j) fb[j] = frag(sb + j * (4 * FP8_BLOCK), rdB);
    if constexpr (std::is_same_v<OT, float>) {
      Wide wb[TN];
#pragma unroll
      for (int j = 0; j < TN; ++j) wb[j] = widen(fb[j]);
#pragma unroll
      for (int i = 0; i < TM; ++i)
        add_block(acc[i], wb, widen(frag(sa + i * (16 * FP8_BLOCK), rdA)), (ea[i / 4] >> (8 * (i % 4))) & 255, eb);
      return;
    }
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const i8v fa = frag(sa + i * (16 * FP8_BLOCK), rdA);
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        // (the byte of the scale register is an immediate of the instruction)
        if (i % 4 == 0) acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[j], fa, acc[i][j], 0, 0, 0, eb, 0, ea[i / 4]);
        else if (i % 4 == 1) acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[j], fa, acc[i][j], 0, 0, 0, eb, 1, ea[i / 4]);
        else if (i % 4 == 2) acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[j], fa, acc[i][j], 0, 0, 0, eb, 2, ea[i / 4]);
        else acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[j], fa, acc[i][j], 0, 0, 0, eb, 3, ea[i / 4]);
      }
    }
  };
  for (int kb = 0; kb < full; ++kb) step(kb, std::false_type{});
  if (krem) step(full, std::true_type{});
  // Output: a lane holds columns 16 q .. 16 q + 15 of row r per tile row.  Exchanging 16-lane rows between two tile rows leaves
  // 32 columns of one row per lane, and a transposition in the quad 64 consecutive bytes per four lanes.
  float bv[TN][4];
#pragma unroll
  for (int j = 0; j < TN; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) bv[j][e] = 0.f;
  if (g.bias) {
    const float *b = g.bias + n0;
    const int left = (int)(g.N - n0 < BN ? g.N - n0 : BN);
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {      // (columns behind the last are not stored: they take its bias, for a branch costs more)
        const int c = wn * (16 * TN) + q * 16 + j * 4 + e;
        bv[j][e] = b[c < left ? c : left - 1];
      }
  }
  if constexpr (std::is_same_v<OT, float>) {      // (fp32: 64 bytes of one row per lane as it is, the transposition alone)
    const int64_t c = n0 + wn * (16 * TN) + q * 16 + (lane & 3) * 4;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      unsigned p[4][4];      // [element][piece of 4 columns]
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) p[e][j] = __float_as_uint(acc[i][j][e] + bv[j][e]);
      quad_transpose4(p);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int64_t m = m0 + wm * (16 * TM) + i * 16 + ((lane >> 2) & 3) * 4 + t;
        if (m < g.M && c < g.N) {
          unsigned *o = (unsigned *)g.C + m * g.ldc + c;
          if (vec && c + 4 <= g.N) {
            *reinterpret_cast<uint4 *>(o) = make_uint4(p[0][t], p[1][t], p[2][t], p[3][t]);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (c + e < g.N) o[e] = p[e][t];
          }
        }
      }
    }
    return;
  }
  const int64_t c = n0 + wn * (16 * TN) + (q >> 1) * 32 + (lane & 3) * 8;
#pragma unroll
  for (int i = 0; i < TM; i += 2) {
    unsigned p[4][4];      // [dword][piece of 8 columns]
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const unsigned a = pack_bf16x2(acc[i][j][2 * w] + bv[j][2 * w], acc[i][j][2 * w + 1] + bv[j][2 * w + 1]);
        const unsigned b = pack_bf16x2(acc[i + 1][j][2 * w] + bv[j][2 * w], acc[i + 1][j][2 * w + 1] + bv[j][2 * w + 1]);
        const auto s = __builtin_amdgcn_permlane16_swap(a, b, false, false);
        p[(j & 1) * 2 + w][j >> 1] = s[0];
        p[(j & 1) * 2 + w][2 + (j >> 1)] = s[1];
      }
    quad_transpose4(p);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int64_t m = m0 + wm * (16 * TM) + (i + (q & 1)) * 16 + ((lane >> 2) & 3) * 4 + t;
      if (m < g.M && c < g.N) {
        bf16_t *o = (bf16_t *)g.C + m * g.ldc + c;
        if (vec && c + 8 <= g.N) {
          *reinterpret_cast<uint4 *>(o) = make_uint4(p[0][t], p[1][t], p[2][t], p[3][t]);
        } else if (vec) {      // (pairs: single elements cost 1000x1111x1000 4 %)
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            if (c + e + 1 < g.N) reinterpret_cast<unsigned *>(o)[e / 2] = p[e / 2][t];
            else if (c + e < g.N) o[e] = (bf16_t)p[e / 2][t];
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (c + e < g.N) o[e] = (bf16_t)(p[e / 2][t] >> (16 * (e & 1)));
        }
      }
    }
  }
}

// workgroups along x: a grid of 2^32 threads and more is cut off without an error
constexpr int64_t MAX_WGS = 0xffffffffll / 256;

template <int TM, typename OT>
int launch_tile(const GArgs &g, hipStream_t s) {
  constexpr int BM = 32 * TM, LDS = 2 * (BM + 128) * FP8_BLOCK + SCH * (BM + 1);
  const int64_t tm = ceil_div(g.M, BM), tn = ceil_div(g.N, 128);
  if (tm > MAX_WGS || tn > MAX_WGS || tm * tn > MAX_WGS) return LDM_E_SHAPE;
  // 32-bit source offsets inside a tile
  if (g.lda >= (1 << 23) || g.ldb >= (1 << 23)) return LDM_E_SHAPE;
  const bool vec = g.ldc % (16 / (int)sizeof(OT)) == 0 && aligned_to(g.C, 16);
  static std::atomic<uint64_t> attr_done{0};
  uint64_t bit;
  if (ldm_attr_pending(attr_done, &bit)) {
    (void)hipFuncSetAttribute((const void *)gemm_fp8_tile_k<TM, OT>, hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
    attr_done.fetch_or(bit, std::memory_order_release);
  }
  hipLaunchKernelGGL((gemm_fp8_tile_k<TM, OT>), dim3((unsigned)(tm * tn)), dim3(256), LDS, s, g, (int)tm, (int)tn, 8, vec);
  LDM_CHECK_LAUNCH();
  return LDM_OK;
}

template <typename OT>
int launch_rows(const GArgs &g, hipStream_t s) {
  const bool vec = g.ldc % 4 == 0 && aligned_to(g.C, 4 * sizeof(OT));
  const int64_t gx = ceil_div(g.N, 16);
  const int mt = g.M <= 16 ? 1 : g.M <= 32 ? 2 : 4;
  const int64_t gy = ceil_div(g.M, 16 * mt);
  if (gx > MAX_WGS || gy > 65535) return LDM_E_SHAPE;
  const dim3 grid((unsigned)gx, (unsigned)gy), wg(256);
  if (mt == 1) hipLaunchKernelGGL((gemm_fp8_rows_k<1, OT>), grid, wg, 0, s, g, vec);
  else if (mt == 2) hipLaunchKernelGGL((gemm_fp8_rows_k<2, OT>), grid, wg, 0, s, g, vec);
  else hipLaunchKernelGGL((gemm_fp8_rows_k<4, OT>), grid, wg, 0, s, g, vec);
  LDM_CHECK_LAUNCH();
  return LDM_OK;
}

int launch_4w(const GArgs &g, hipStream_t s) {
  return ldm_gemm_fp8_4w(g.M, g.N, g.K, g.A, g.lda, g.sA, g.ld_sa, g.B, g.ldb, g.sB, g.ld_sb, g.C, g.ldc, g.bias, s);
}

constexpr int64_t CUS = 256;

// Tile height by rounds of what is resident: two 128 x 128 tiles per CU, or three of 64 x 128; the smaller ones where they need no
// more rounds (us at 64 / 128 rows: 2048x2304x768, one round each, 9.9 / 10.1; 2048x768x768 5.6 / 7.5; 4096x2304x768, two each,
// 15.4 / 16.7; 8192x2304x768, three each, 25.7 / 25.7; 3000x2304x768, two against one, 14.5 / 11.1; 256x30522x768 15.1 / 12.8;
// 512x30522x768, three against two, 23.7 / 22.3; 777x30522x768 34.5 / 33.5; 4096x2048x2048 26.8 / 19.6).
template <typename OT>
int launch_tiles(const GArgs &g, hipStream_t s) {
  const int64_t tn = ceil_div(g.N, 128);
  const bool low = ceil_div(ceil_div(g.M, 64) * tn, 3 * CUS) <= ceil_div(ceil_div(g.M, 128) * tn, 2 * CUS);
  const int rc = low ? launch_tile<2, OT>(g, s) : launch_tile<4, OT>(g, s);
  return rc == LDM_E_SHAPE ? launch_rows<OT>(g, s) : rc;      // (row strides of 8 MiB and more)
}

GArgs columns_from(const GArgs &g, int64_t n) {      // bf16 output; n: a multiple of 128
  GArgs t = g;
  t.N = g.N - n;
  t.B += n * g.ldb;
  t.sB += n / FP8_BLOCK * g.ld_sb;
  t.C = (bf16_t *)g.C + n;
  if (t.bias) t.bias += n;
  return t;
}

// Which kernel, by what was measured (us, both sides):
//   few rows: the row kernel while its workgroups are about one per CU (64x2304x768 4.3 against 5.1 for 64 x 128 tiles,
//     256x768x768 4.3 / 5.1, 96x2304x768 5.3 / 5.1, 512x768x768 6.0 / 5.2, 64x11264x2048 18.9 / 12.4), up to 32 rows four per CU
//     (32x11264x2048 12.0 / 12.3, 32x30522x768 11.8 / 8.2), up to 16 always (16x11264x2048 8.5 / 12.2, 16x30522x768 8.3 / 8.1);
//   four waves per 256 x 256 tile when the outputs fill three quarters of its rounds of 256 workgroups (4096x4096x768: one
//     round 19.3 against 21.8 for 128 x 128 tiles; 16384x2304x768: 0.75 of 3 rounds 44.7 / 46.9; 1536x8192x768: 0.75 of one
//     18.0 / 17.8; 15001x2304x768: 0.69 of 3 44.5 / 41.8; 8192x2304x768: 0.56 of 2 28.8 / 25.7; 4096x11264x2048: 0.92 of 3
//     88 / 119).  Columns behind the last multiple of 128 are a second launch: it pays where the first one saves more
//     (1024x30522x768: 0.93 of 2 44.3 / 46.0; 15001x11200x768: 0.91 of 11 184 / 186).
//   fp32 output has rows and tiles: rows up to two workgroups per CU (64 x 128 tiles: 96x2304x768 5.9 / 8.7, 512x768x768 6.6 /
//     8.7, 64x11264x2048 18.5 / 16.8, 2048x768x768 16.7 / 9.3; up to 32 rows 32x11264x2048 11.4 / 16.2, 32x30522x768 11.9 / 8.8;
//     16x30522x768 8.0 / 8.1), and the same choice of tile height (64 / 128 rows: 2048x2304x768 17.0 / 20.1, 3000x2304x768 21.9 /
//     20.5, 8192x2304x768 43.5 / 43.7, 512x30522x768 39.0 / 36.5, 777x30522x768 59.0 / 58.2).  16384x11264x2048 768 us = 985
//     TFLOP/s; 777x30522x768 62 us, of which the matrix pipe is busy 25 % and vector instructions (widening, ldexp, additions,
//     packing) issue in 44 %: the two do not overlap among a SIMD's waves on this card, and six steps of K leave the rest to
//     waits and stores.
template <typename OT>
int launch(const GArgs &g, hipStream_t s) {
  const int64_t gx = ceil_div(g.N, 16);
  constexpr int64_t FEW = std::is_same_v<OT, float> ? 2 * CUS : CUS;
  if (g.M <= 16 || gx * ceil_div(g.M, 64) <= (g.M <= 32 ? 4 * CUS : FEW)) return launch_rows<OT>(g, s);
  if constexpr (std::is_same_v<OT, float>) return launch_tiles<OT>(g, s);
  const int64_t n128 = g.N / FP8_BLOCK * FP8_BLOCK;
  const int64_t rounds = ceil_div(ceil_div(g.M, 256) * ceil_div(n128, 256), CUS);
  if ((double)g.M * (double)n128 >= (n128 == g.N ? 0.75 : 0.85) * 65536.0 * (double)(rounds * CUS)) {
    GArgs m = g;
    m.N = n128;
    const int rc = launch_4w(m, s);
    if (rc != LDM_E_SHAPE && rc != LDM_E_ALIGN) return rc != LDM_OK || n128 == g.N ? rc : launch_tiles<OT>(columns_from(g, n128), s);
  }
  return launch_tiles<OT>(g, s);
}

// checks of the C entries; elt: bytes of an output element
int checked(const GArgs &g, int elt) {
  if (g.M < 0 || g.N < 0 || g.K <= 0) return LDM_E_BADARG;
  if (g.M == 0 || g.N == 0) return LDM_OK;
  if (!g.A || !g.sA || !g.B || !g.sB || !g.C) return LDM_E_BADARG;
  const int64_t kb = ceil_div(g.K, FP8_BLOCK);
  if (g.lda < g.K || g.ldb < g.K || g.ldc < g.N || g.ld_sa < kb || g.ld_sb < kb) return LDM_E_BADARG;
  if (g.lda % 16 || g.ldb % 16 || !aligned_to(g.A, 16) || !aligned_to(g.B, 16)) return LDM_E_ALIGN;
  if (!aligned_to(g.C, elt) || (g.bias && !aligned_to(g.bias, 4))) return LDM_E_ALIGN;
  if (g.M > (1ll << 40) || g.N > (1ll << 31) || g.K > (1 << 28)) return LDM_E_SHAPE;
  return LDM_OK;
}

}  // namespace

extern "C" int ldm_gemm_fp8(int64_t M, int64_t N, int64_t K, const uint8_t *A, int64_t lda, const uint8_t *sA,
                            int64_t ld_sa, const uint8_t *B, int64_t ldb, const uint8_t *sB, int64_t ld_sb,
                            const float *bias, void *C, int64_t ldc, void *stream) {
  const GArgs g{M, N, K, A, lda, sA, ld_sa, B, ldb, sB, ld_sb, bias, C, ldc};
  const int rc = checked(g, 2);
  return rc != LDM_OK || M == 0 || N == 0 ? rc : launch<bf16_t>(g, (hipStream_t)stream);
}

extern "C" int ldm_gemm_fp8_f32(int64_t M, int64_t N, int64_t K, const uint8_t *A, int64_t lda, const uint8_t *sA,
                                int64_t ld_sa, const uint8_t *B, int64_t ldb, const uint8_t *sB, int64_t ld_sb,
                                const float *bias, float *C, int64_t ldc, void *stream) {
  const GArgs g{M, N, K, A, lda, sA, ld_sa, B, ldb, sB, ld_sb, bias, C, ldc};
  const int rc = checked(g, 4);
  return rc != LDM_OK || M == 0 || N == 0 ? rc : launch<float>(g, (hipStream_t)stream);
}
