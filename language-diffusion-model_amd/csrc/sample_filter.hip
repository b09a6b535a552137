// Token choice from given random numbers with temperature, top-k, top-p and min-p (inference).
//
// A row's weights are w_i = exp((l_i - max l) / temperature).  Tokens are ordered by (logit descending, index ascending);
// the kept set is a prefix of that order: at most top_k tokens, the shortest prefix that reaches top_p of the weight of the
// top_k, and no token below min_p (the largest weight is 1).  The choice inverts the distribution function of the kept
// tokens in INDEX order: the first i with sum_{kept j <= i} w_j > u * sum_kept w.  So nothing is ever sorted: each
// filter only has to find its cut, the last kept (logit, index) pair.
//
// Weights are 64-bit integers, round(w * 2^shift): their sums do not depend on the order they are formed in (LDS atomics,
// any number of waves), so the same row gives the same token every time, and a border is decided by at most 2^-shift of
// the largest weight per token.
//
// One workgroup per row.  Passes over the row (the first from memory, the others mostly from the caches):
//   1. largest and smallest logit;
//   2. a histogram of counts (top_k) or of estimated weights (top_p) over max - logit, linear bins, monotone in the logit; a scan
//      finds the bin of the cut;
//   3. the tokens of that bin are listed and ranked exactly against each other, while the exact weights in front of it are
//      summed per 1024-token segment; the ranked tokens that stay are added, and a scan finds the segment of the choice.
// The exact sums of pass 3 also tell whether the estimates had found the right bin (off by 1e-6 of the sum, it is wrong
// for about one row in a thousand); if not, the histogram is repeated with the integer weights.  With top_k and top_p both,
// pass 3 lists everything down to the bin (top_k tokens and the rest of one bin) and the weights' histogram, ranking and
// sums run on the list.  Where more tokens share the cut's
// bin than the list holds, a second histogram divides that bin, equal logits are counted by index, and only thousands of
// different logits within 1e-7 of the range are bisected.
//
// Bound by the vector unit while a pass runs (about 20 double operations per weight) and by the barriers, scans and ranking
// between the passes: 1000 rows of 126464 fp32 logits 325 us (1.6 TB/s of the row read once; 60 % of the cycles issue vector
// instructions), 2048 rows of 30522 bf16 114 us (1.1 TB/s; 38 %), 32 rows 30 us, the time of one.

#include <limits.h>

#include "common.h"

namespace {

constexpr int SEG = 1024;         // tokens per segment of the final distribution function (one wave, 2 x 8 each)
constexpr int MAX_V = 262144;
typedef unsigned long long u64;

struct FArgs {
  int64_t ld;
  int V;
  const float *u;
  const int64_t *ids;      // nullable
  int64_t mask_id;
  double inv_temp, top_p, min_p;
  int top_k;               // 0: off
  int shift;
  int64_t *out;
};

struct alignas(16) Token { float v; int i; u64 w; };      // logit, index, weight

// NT: threads per row; NB: histogram bins
template <int NT, int NB>
struct Shared {
  static constexpr int BCAP = NB / 4 < 256 ? 256 : NB / 4;      // tokens around the cut that are ranked exactly
  static constexpr int LCAP = NB / 2;                   // tokens down to the top_k cut's bin that are kept as a list
  u64 hist[NB];
  Token bt[BCAP + 4];
  float lv[LCAP];
  int li[LCAP];
  u64 seg[NB <= 1024 ? 8 : MAX_V / SEG];                // (V <= 1024 has one segment, V <= 8192 eight)
  u64 red[NT / 64], red2[NT / 64];
  float redf[NT / 64], redg[NT / 64];
  u64 base;                // measure in front of the cut's bin
  int bin, bin_lo, bin_hi; // the cut's bin, and the bins (lo .. hi) it may be in if the histogram holds estimates
  int nbin, nlist, rank;
  float cut_v;
  int cut_i;
};

// eight consecutive logits at any element alignment; NaN behind the last one
struct __attribute__((packed, aligned(2))) u4a2 { unsigned w[4]; };
struct __attribute__((packed, aligned(4))) f4a4 { float w[4]; };
__device__ __forceinline__ void load8(const bf16_t *row, int c, int V, float (&x)[8]) {
  if (c >= V) {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = __builtin_nanf("");
  } else if (c + 8 <= V) {
    const u4a2 t = *reinterpret_cast<const u4a2 *>(row + c);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[2 * j] = __uint_as_float(t.w[j] << 16);
      x[2 * j + 1] = __uint_as_float(t.w[j] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = c + j < V ? bf16_to_f32(row[c + j]) : __builtin_nanf("");
  }
}
__device__ __forceinline__ void load8(const float *row, int c, int V, float (&x)[8]) {
  if (c >= V) {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = __builtin_nanf("");
  } else if (c + 8 <= V) {
    const f4a4 a = *reinterpret_cast<const f4a4 *>(row + c), b = *reinterpret_cast<const f4a4 *>(row + c + 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) { x[j] = a.w[j]; x[4 + j] = b.w[j]; }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = c + j < V ? row[c + j] : __builtin_nanf("");
  }
}

__device__ __forceinline__ u64 wave_sum_u64(u64 v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
__device__ __forceinline__ u64 wave_scan_u64(u64 v) {      // inclusive
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const u64 t = __shfl_up(v, o, 64);
    if (lane >= o) v += t;
  }
  return v;
}
// sum over the workgroup, the same value in every thread (two barriers)
template <int NT, int NB>
__device__ __forceinline__ u64 block_sum(u64 v, Shared<NT, NB> &s) {
  v = wave_sum_u64(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s.red[threadIdx.x >> 6] = v;
  __syncthreads();
  u64 t = 0;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) t += s.red[i];
  return t;
}

struct Row {
  float mx;
  float bin_scale, bin_last;
  float floor;       // every logit at and below it has weight 0 and is taken as this
  float cf;          // log2(e) / temperature
  double dmx, c;     // mx; log2(e) / temperature
  int shift;
  // round(2^shift * 2^-x), x = c (mx - l) >= 0 and at most about 2 (shift + 3) (logits are held to `floor`, where the weight is
  // 0): 2^-n times a polynomial for 2^f on |f| <= 1/2 (degree 9 through the Chebyshev nodes, constant term 1: off by
  // 3e-14).  n comes out of adding 1.5 * 2^52, the power of two goes into the exponent bits, and the integer out of adding
  // 2^52: the conversions, roundings and scalings of doubles that the card has run at a quarter of the rate of these sums.
  __device__ __forceinline__ double weight_d(float l) const {      // as a double
    const double x = (dmx - (double)l) * c;
    const double nm = x + 6755399441055744.0;
    const double f = (nm - 6755399441055744.0) - x;
    double p = 1.0205905413765595e-07;
    p = fma(p, f, 1.325964524488711e-06);
    p = fma(p, f, 1.5252672924850737e-05);
    p = fma(p, f, 1.540343375125101e-04);
    p = fma(p, f, 1.3333558200794592e-03);
    p = fma(p, f, 9.618129193934313e-03);
    p = fma(p, f, 5.550410866465167e-02);
    p = fma(p, f, 2.402265069564034e-01);
    p = fma(p, f, 6.931471805599462e-01);
    p = fma(p, f, 1.0);
    const int n = __double2loint(nm);
    const double t = __hiloint2double(__double2hiint(p) + ((shift - n) << 20), __double2loint(p)) + 4503599627370496.0;
    return t - 4503599627370496.0;
  }
  __device__ __forceinline__ u64 weight(float l) const { return (u64)weight_d(l); }
  // an estimate from the fp32 exponential, in units of 2^-32, only to find a bin.  (Integers all the same: a float addition
  // in LDS takes its lanes one by one, 190 cycles an instruction against about 20 for the 64-bit integer.)
  __device__ __forceinline__ u64 estimate(float l) const { return (unsigned)fmaf(__builtin_amdgcn_exp2f((l - mx) * cf), 4294967040.f, 0.5f); }
  // max(v, floor), floor for a NaN: the median with +infinity (a maximum costs a second instruction to quiet NaNs)
  __device__ __forceinline__ float hold(float v) const { return __builtin_amdgcn_fmed3f(v, floor, INFINITY); }
  __device__ __forceinline__ float bin_f(float l) const { return fminf((mx - l) * bin_scale, bin_last); }     // its integer part
  __device__ __forceinline__ int bin(float l) const { return (int)bin_f(l); }
};

// monotone unsigned key of a float (no NaN)
__device__ __forceinline__ unsigned fkey(float f) {
  f = f == 0.f ? 0.f : f;      // -0 and +0 are equal logits
  const unsigned b = __float_as_uint(f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float fkey_inv(unsigned k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

struct Cut { float v; int i; };
__device__ __forceinline__ bool kept(const Cut &c, float l, int i) { return l > c.v || (l == c.v && i <= c.i); }

// f(logit, index) for every token of the row this thread owns: a wave has 1024 consecutive ones, 2 x 8 per lane.  Logits
// without weight (NaN, -infinity, everything below `floor`, and what lies behind the last token) come as `floor`.
template <int NT, typename T, typename F>
__device__ __forceinline__ void each_of_row(const T *row, int V, const Row &rw, F f) {
  for (int c = (threadIdx.x >> 6) * SEG + (threadIdx.x & 63) * 8; c < V; c += NT * 16) {
    float x[2][8];
#pragma unroll
    for (int u = 0; u < 2; ++u) load8(row, c + u * 512, V, x[u]);
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int j = 0; j < 8; ++j) f(rw.hold(x[u][j]), c + u * 512 + j);
  }
}
// the same with smaller code, for what rarely runs
template <int NT, typename T, typename F>
__device__ __forceinline__ void each_of_row_slowly(const T *row, int V, const Row &rw, F f) {
#pragma unroll 1
  for (int c = threadIdx.x * 8; c < V; c += NT * 8) {
    float x[8];
    load8(row, c, V, x);
#pragma unroll
    for (int j = 0; j < 8; ++j) f(rw.hold(x[j]), c + j);
  }
}
template <int NT, int NB, typename F>
__device__ __forceinline__ void each_of_list(const Shared<NT, NB> &s, int n, F f) {
  for (int t = threadIdx.x; t < n; t += NT) f(s.lv[t], s.li[t]);
}

template <int NT, int NB>
__device__ __forceinline__ void clear_hist(Shared<NT, NB> &s) {
  __syncthreads();
  for (int b = threadIdx.x; b < NB; b += NT) s.hist[b] = 0;
  if (threadIdx.x == 0) { s.nbin = 0; s.nlist = 0; s.rank = -1; s.bin = s.bin_lo = s.bin_hi = -1; }
  __syncthreads();
}

// sums are integers: before < target as before < ceil(target), after > target as after > floor(target)
__device__ __forceinline__ u64 share_of(double share, u64 total) { return (u64)ceil(share * (double)total); }

// The bin where "measure in front < target" ends: s.bin (-1: the target is not reached) and s.base.  A few bins per thread,
// then a scan over the threads.  `first`: what lies in front of the histogram.  SHARE: the target is a share of its sum.
// Returns the target.
template <bool SHARE, int NT, int NB>
__device__ __forceinline__ u64 find_bin(double share, u64 target, u64 first, Shared<NT, NB> &s) {
  __syncthreads();
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  constexpr int per = NB / NT;
  u64 sum = 0;
  for (int j = 0; j < per; ++j) sum += s.hist[threadIdx.x * per + j];
  const u64 inc = wave_scan_u64(sum);
  if (lane == 63) s.red[wid] = inc;
  __syncthreads();
  u64 before = first + inc - sum, total = 0;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) {
    const u64 r = s.red[w];
    before += w < wid ? r : 0ull;
    total += r;
  }
  if (SHARE) target = share_of(share, total);
  if (before < target && before + sum >= target) {      // (one thread, if any)
    for (int j = 0; j < per; ++j) {
      const u64 h = s.hist[threadIdx.x * per + j];
      if (before < target && before + h >= target) {
        const int b = threadIdx.x * per + j;
        s.bin = b;
        s.base = before;
        // (estimates are off by about 1e-5 of the sum: near an edge of the bin its neighbour is taken in)
        const u64 edge = SHARE ? total >> 15 : 0;
        s.bin_lo = target - before <= edge && b > 0 ? b - 1 : b;
        s.bin_hi = before + h - target <= edge && b < NB - 1 ? b + 1 : b;
      }
      before += h;
    }
  }
  __syncthreads();
  return target;
}

template <int NT, int NB>
__device__ __forceinline__ void add_to_bin(Shared<NT, NB> &s, float v, int i, u64 w) {
  const int p = atomicAdd(&s.nbin, 1);
  if (p < s.BCAP) s.bt[p] = Token{v, i, w};
}

// Lists every token of the row with weight in the bins up to `bin`; returns their number (more than s.LCAP: the list is cut off).
// BINS: those of the bin itself go to its own list as well.
template <bool BINS, typename T, int NT, int NB>
__device__ __forceinline__ int list_down_to(const T *row, int V, const Row &rw, int bin, Shared<NT, NB> &s) {
  const float hi = (float)(bin + 1);
  for (int c = (threadIdx.x >> 6) * SEG + (threadIdx.x & 63) * 8; c < V; c += NT * 16) {
    float x[2][8];
#pragma unroll
    for (int h = 0; h < 2; ++h) load8(row, c + h * 512, V, x[h]);
    unsigned hits = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float l = rw.hold(x[h][j]);
        hits |= rw.bin_f(l) < hi && l > rw.floor ? 1u << (h * 8 + j) : 0u;      // (never behind the last token)
      }
    while (hits) {
      const int k = __ffs(hits) - 1, i = c + (k >> 3) * 512 + (k & 7);
      const int p = atomicAdd(&s.nlist, 1);
      const float l = rw.hold(Elt<T>::ld(row + i));
      if (p < s.LCAP) { s.lv[p] = l; s.li[p] = i; }
      if (BINS && rw.bin(l) == bin) add_to_bin(s, l, i, 1ull);
      hits &= hits - 1;
    }
  }
  __syncthreads();
  return s.nlist;
}

// Exact cut among the n <= BCAP listed tokens of the bin: kept while the measure in front is below the target (at least one
// is).  After it every thread has the cut.
template <bool WEIGHT, int NT, int NB>
__device__ __forceinline__ Cut rank_bin(int n, u64 target, Shared<NT, NB> &s) {
  // every pair of tokens is compared once: `parts` threads share a token's comparisons where there are threads to spare, and
  // add up in the histogram's memory (first half: measure in front, second half: rank)
  const int stride = (n + 63) & ~63;
  const int parts = stride < NT ? NT / stride : 1;
  const int chunk = ((n + parts - 1) / parts + 3) & ~3;
  u64 *measure = s.hist, *ranks = s.hist + s.BCAP;
  __syncthreads();
  for (int c = threadIdx.x; c < n; c += NT) measure[c] = ranks[c] = 0;
  if (threadIdx.x < 4) s.bt[n + threadIdx.x] = Token{-INFINITY, INT_MAX, 0ull};      // the loop takes four at a time
  __syncthreads();
  const int part = parts > 1 ? threadIdx.x / stride : 0;
  for (int c = parts > 1 ? threadIdx.x - part * stride : threadIdx.x; c < n && part < parts; c += parts > 1 ? n : NT) {
    const Cut me{s.bt[c].v, s.bt[c].i};
    const int end = (part + 1) * chunk < n ? (part + 1) * chunk : n;
    u64 before = 0;
    int r = 0;
    for (int j = part * chunk; j < end; j += 4) {
      Token t[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) t[k] = s.bt[j + k];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const bool pre = t[k].v > me.v || (t[k].v == me.v && t[k].i < me.i);
        if (WEIGHT) before += pre ? t[k].w : 0ull;
        r += pre ? 1 : 0;
      }
    }
    if (r) {
      if (WEIGHT) atomicAdd(&measure[c], before);
      atomicAdd(&ranks[c], (u64)r);
    }
  }
  __syncthreads();
  int best = -1;
  Cut mine{0.f, 0};
  for (int c = threadIdx.x; c < n; c += NT) {
    const int r = (int)ranks[c];
    const u64 before = s.base + (WEIGHT ? measure[c] : (u64)r);
    if (before < target && r > best) { best = r; mine = Cut{s.bt[c].v, s.bt[c].i}; }
  }
  if (best >= 0) atomicMax(&s.rank, best);
  __syncthreads();
  if (best >= 0 && best == s.rank) { s.cut_v = mine.v; s.cut_i = mine.i; }
  __syncthreads();
  return Cut{s.cut_v, s.cut_i};
}

// The same cut by bisection, for a bin with more tokens than the list holds.
template <bool WEIGHT, typename T, int NT, int NB>
__device__ __forceinline__ Cut bisect(const T *row, int V, const Row &rw, const Cut &cur, u64 target, Shared<NT, NB> &s) {
  unsigned lo = 0, hi = fkey(rw.mx);             // the smallest key K with measure{key > K} < target; measure{key > hi} = 0
  u64 front = 0;
  while (lo < hi) {
    const unsigned mid = lo + (hi - lo) / 2;
    u64 m = 0;
    each_of_row_slowly<NT>(row, V, rw, [&](float l, int i) { if (fkey(l) > mid && l > rw.floor && kept(cur, l, i)) m += WEIGHT ? rw.weight(l) : 1ull; });
    m = block_sum(m, s);
    if (m < target) { hi = mid; front = m; } else lo = mid + 1;
  }
  const float v = fkey_inv(lo);
  const u64 w = WEIGHT ? rw.weight(v) : 1ull;
  int ilo = 0, ihi = V - 1;                      // the last index whose equals in front leave the measure below the target
  while (ilo < ihi) {
    const int mid = ilo + (ihi - ilo + 1) / 2;
    u64 m = 0;
    each_of_row_slowly<NT>(row, V, rw, [&](float l, int i) { if (i < mid && l == v && kept(cur, l, i)) m += w; });
    m = block_sum(m, s);
    if (front + m < target) ilo = mid; else ihi = mid - 1;
  }
  return (v > cur.v || (v == cur.v && ilo < cur.i)) ? Cut{v, ilo} : cur;
}

// The cut among the tokens of the bins lo .. hi, of which there are more than the list holds; `front` is the measure in front
// of them.  A second histogram inside these bins, then the list again; where the values themselves are equal, a histogram
// over the index; what is left (thousands of different values within 1e-7 of the range) is bisected.  false: the target
// is not reached inside.
template <bool WEIGHT, typename T, int NT, int NB>
__device__ __forceinline__ bool refine(const T *row, int V, const Row &rw, Cut &cut, int lo, int hi, u64 front, u64 target,
                                       Shared<NT, NB> &s) {
  const Cut cur = cut;
  const float flo = (float)lo, fhi = (float)(hi + 1), scale = (float)NB / (fhi - flo);
  auto sub = [&](float t) { return (int)fminf((t - flo) * scale, (float)(NB - 1)); };
  auto inside = [&](float l, float t, int i) { return t >= flo && t < fhi && l > rw.floor && kept(cur, l, i); };
  clear_hist(s);
  each_of_row_slowly<NT>(row, V, rw, [&](float l, int i) {
    const float t = rw.bin_f(l);
    if (inside(l, t, i)) atomicAdd(&s.hist[sub(t)], WEIGHT ? rw.weight(l) : 1ull);
  });
  find_bin<false>(0.0, target, front, s);
  const int sb = s.bin;
  if (sb < 0) return false;
  const u64 base = s.base;
  float mn = INFINITY, mx = -INFINITY;
  each_of_row_slowly<NT>(row, V, rw, [&](float l, int i) {
    const float t = rw.bin_f(l);
    if (inside(l, t, i) && sub(t) == sb) {
      add_to_bin(s, l, i, WEIGHT ? rw.weight(l) : 1ull);
      mn = fminf(mn, l);
      mx = fmaxf(mx, l);
    }
  });
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    mx = fmaxf(mx, __shfl_xor(mx, o, 64));
    mn = fminf(mn, __shfl_xor(mn, o, 64));
  }
  if ((threadIdx.x & 63) == 0) { s.redf[threadIdx.x >> 6] = mx; s.redg[threadIdx.x >> 6] = mn; }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) { mx = fmaxf(mx, s.redf[i]); mn = fminf(mn, s.redg[i]); }
  const int n = s.nbin;
  if (n <= s.BCAP) {
    cut = rank_bin<WEIGHT>(n, target, s);
    return true;
  }
  if (mn < mx) {
    cut = bisect<WEIGHT>(row, V, rw, cur, target, s);
    return true;
  }
  // equal values: as many of the lowest indexes as the target takes
  const u64 w = WEIGHT ? rw.weight(mx) : 1ull;
  const u64 count = (target - base + w - 1) / w;
  const int width = (V + NB - 1) / NB;
  clear_hist(s);
  each_of_row_slowly<NT>(row, V, rw, [&](float l, int i) { if (l == mx && kept(cur, l, i)) atomicAdd(&s.hist[i / width], 1ull); });
  find_bin<false>(0.0, count, 0ull, s);
  const int ib = s.bin;
  each_of_row_slowly<NT>(row, V, rw, [&](float l, int i) { if (l == mx && i / width == ib && kept(cur, l, i)) add_to_bin(s, l, i, 1ull); });
  __syncthreads();
  cut = rank_bin<false>(s.nbin, count, s);
  return true;
}

// Exact weights of the kept tokens per segment.  BIN: only those in front of the bins bin_lo .. bin_hi, whose tokens go to the list,
// and every thread gets the weight in front of it (before min_p) and of everything.  GEN: apply the cut and min_p.
template <bool BIN, bool GEN, typename T, int NT, int NB>
__device__ __forceinline__ void sum_segments(const T *row, int V, const Row &rw, const Cut &cut, double wmin, int bin_lo, int bin_hi,
                                             Shared<NT, NB> &s, u64 &front, u64 &total) {
  u64 fr = 0, tot = 0;
  const float lo = (float)bin_lo, hi = (float)(bin_hi + 1);
  // (a wave's lanes stay together to its last segment, for they add up there; what is behind the row weighs nothing)
  for (int c0 = (threadIdx.x >> 6) * SEG; c0 < V; c0 += NT * 16) {
    const int c = c0 + (threadIdx.x & 63) * 8;
    float x[2][8];
#pragma unroll
    for (int u = 0; u < 2; ++u) load8(row, c + u * 512, V, x[u]);
    // (sums of 16 integers of at most 2^45 are exact in a double)
    double m = 0.0, f = 0.0, t = 0.0;
    unsigned hits = 0;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float l = rw.hold(x[u][j]);
        double w = rw.weight_d(l);
        if (GEN) w = kept(cut, l, c + u * 512 + j) ? w : 0.0;
        if (BIN) {
          const float b = rw.bin_f(l);
          t += w;
          hits |= b >= lo && b < hi && l > rw.floor ? 1u << (u * 8 + j) : 0u;      // (never behind the last token)
          w = b < lo ? w : 0.0;
          f += w;
        }
        if (GEN) w = w >= wmin ? w : 0.0;
        if (GEN || !BIN) m += w;
      }
    // (out of the unrolled part: a branch per token there costs more than the weights)
    while (BIN && hits) {
      const int k = __ffs(hits) - 1, i = c + (k >> 3) * 512 + (k & 7);
      const float l = rw.hold(Elt<T>::ld(row + i));
      const u64 w = rw.weight(l);
      if (w && (!GEN || kept(cut, l, i))) add_to_bin(s, l, i, w);
      hits &= hits - 1;
    }
    const u64 seg = wave_sum_u64((u64)(GEN || !BIN ? m : f));
    if ((threadIdx.x & 63) == 0) s.seg[c0 / SEG] = seg;
    fr += (u64)f;
    tot += (u64)t;
  }
  if (BIN) {
    fr = wave_sum_u64(fr);
    tot = wave_sum_u64(tot);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) { s.red[threadIdx.x >> 6] = fr; s.red2[threadIdx.x >> 6] = tot; }
    __syncthreads();
    front = total = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) { front += s.red[w]; total += s.red2[w]; }
  } else {
    __syncthreads();
  }
}

// A row where only the tokens at the largest logit have weight, in equal shares: an infinite logit, a temperature below the
// logits' resolution, a row that is the type's lowest value throughout.  The first wave.
template <typename T>
__device__ __forceinline__ int choose_equal(const T *row, const FArgs &a, float mx, float uf) {
  const int lane = threadIdx.x & 63;
  int n = 0, got = 0, tok = 0;
  double j = 0.0;
  for (int pass = 0; pass < 2; ++pass) {
    for (int c0 = 0; c0 < a.V; c0 += 512) {
      float x[8];
      load8(row, c0 + lane * 8, a.V, x);
      int m = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) m += x[k] == mx ? 1 : 0;
      int inc = m;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int t = __shfl_up(inc, o, 64);
        if (lane >= o) inc += t;
      }
      if (pass == 0) {
        n += __shfl(inc, 63, 64);
        continue;
      }
      int r = got + inc - m;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (x[k] == mx) {
          if ((double)r == j) tok = c0 + lane * 8 + k;
          ++r;
        }
      }
      got += __shfl(inc, 63, 64);
    }
    if (pass == 0) {
      double keep = a.top_k > 0 && a.top_k < n ? (double)a.top_k : (double)n;
      if (a.top_p < 1.0) keep = fmin(keep, ceil(a.top_p * keep));
      double u = (double)uf;
      u = u >= 0.0 ? fmin(u, 0.99999999999999989) : 0.0;
      j = fmin(floor(u * keep), keep - 1.0);
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) tok = max(tok, __shfl_xor(tok, o, 64));
  return tok;
}

// The choice inside a segment's tokens, sorted by index over the lanes: lane's k-th token has weight w[k], index i[k]
// (-1: none).  `before`: weight of the segments in front.  The first wave only.
template <int K>
__device__ __forceinline__ void choose_in_segment(const u64 (&w)[K], const int (&idx)[K], u64 before, u64 target, int64_t *out) {
  u64 m = 0;
#pragma unroll
  for (int j = 0; j < K; ++j) m += w[j];
  u64 cum = before + wave_scan_u64(m) - m;
  int tok = -1;
#pragma unroll
  for (int j = 0; j < K; ++j) {
    cum += w[j];
    if (tok < 0 && w[j] > 0 && cum > target) tok = idx[j];
  }
  const u64 hit = __ballot(tok >= 0);
  if ((int)(threadIdx.x & 63) == (hit ? __ffsll(hit) - 1 : 0)) out[0] = hit ? tok : 0;
}

// Segment of the choice from s.seg: its number, and the weight in front of it (the first wave only; after a barrier).
template <int NT, int NB>
__device__ __forceinline__ int find_segment(int nseg, float uf, u64 &before, u64 &target, Shared<NT, NB> &s) {
  const int lane = threadIdx.x & 63;
  u64 total = 0;
  for (int g = lane; g < nseg; g += 64) total += s.seg[g];
  total = wave_sum_u64(total);
  double u = (double)uf;
  u = u >= 0.0 ? fmin(u, 0.99999999999999989) : 0.0;      // outside [0, 1) or NaN: the nearest choice
  target = (u64)(u * (double)total);
  before = 0;
  for (int g0 = 0; g0 < nseg; g0 += 64) {
    const u64 mine = g0 + lane < nseg ? s.seg[g0 + lane] : 0ull;
    const u64 inc = wave_scan_u64(mine);
    const u64 hit = __ballot(before + inc > target);
    if (hit) {
      const int l = __ffsll(hit) - 1;
      before += __shfl(inc - mine, l, 64);
      return g0 + l;
    }
    before += __shfl(inc, 63, 64);
  }
  return nseg - 1;
}

template <int NT, int NB, typename T>
__global__ __launch_bounds__(NT, 4) void sample_filtered_k(const T *logits, FArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  Shared<NT, NB> &s = *reinterpret_cast<Shared<NT, NB> *>(smem);
  const int64_t r = blockIdx.x;
  if (a.ids) {
    const int64_t id = a.ids[r];
    if (id != a.mask_id) {
      if (threadIdx.x == 0) a.out[r] = id;
      return;
    }
  }
  const T *row = logits + r * a.ld;
  const int V = a.V, lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  float mx = -INFINITY, mn = INFINITY;
  constexpr int U = 4;      // the pass from memory: loads in flight per thread
  for (int c = threadIdx.x * 8; c < V; c += NT * 8 * U) {
    float x[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u) load8(row, c + u * (NT * 8), V, x[u]);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < 8; ++j) {      // (a NaN is neither larger nor smaller)
        mx = fmaxf(mx, x[u][j]);
        mn = fminf(mn, x[u][j]);
      }
  }
  const float own = mx;         // the largest logit this thread has seen
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    mx = fmaxf(mx, __shfl_xor(mx, o, 64));
    mn = fminf(mn, __shfl_xor(mn, o, 64));
  }
  if (lane == 0) { s.redf[wid] = mx; s.redg[wid] = mn; }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) { mx = fmaxf(mx, s.redf[i]); mn = fminf(mn, s.redg[i]); }
  if (mx == -INFINITY) {        // nothing can be chosen: token 0
    if (threadIdx.x == 0) a.out[r] = 0;
    return;
  }
  // Logits at and below it have weight 0 (ln 2 < 0.7): masked places and what lies behind the row stand there.  Where `vanish` is
  // a few steps of mx the subtraction may round towards mx, and half a step leaves a weight: then the next lower float.
  // Temperatures are within 1e-28 .. 1e28, so it is either finite and at least half a step of mx away, or mx itself
  const float vanish = (float)(0.7 * (a.shift + 3) / a.inv_temp);
  float floor = mx < INFINITY ? fmaxf(mx - vanish, -3.402823466e38f) : mx;
  if (floor != mx && mx - floor < vanish) floor = fmaxf(nextafterf(floor, -INFINITY), -3.402823466e38f);
  if (floor == mx) {
    if (wid == 0) {
      const int tok = choose_equal(row, a, mx, a.u[r]);
      if (lane == 0) a.out[r] = tok;
    }
    return;
  }
  Row rw;
  rw.mx = mx;
  rw.c = a.inv_temp * 1.4426950408889634;
  rw.cf = (float)rw.c;
  rw.shift = a.shift;
  rw.dmx = (double)mx;
  rw.floor = floor;
  {
    // bins reach down to the smallest logit or to where weights vanish, whichever is nearer
    const float reach = fminf(mx - mn, mx - floor);
    rw.bin_last = (float)(NB - 1);
    rw.bin_scale = reach > 0.f ? (float)NB / reach : 0.f;
  }
  const double wmin = ceil(a.min_p * (double)(1ull << a.shift));
  const int nseg = (V + SEG - 1) / SEG;
  Cut cut{-INFINITY, INT_MAX};
  bool listed = false;            // the kept tokens are those of s.lv / s.li that pass the cut
  int nlist = 0;

  if (a.top_k > 0) {
    // The top_k-th largest of the threads' own maxima is a lower bound for the top_k-th largest logit, and a near one: where
    // there are enough threads, everything down to its bin is listed, and the cut is found in the list.
    if (a.top_k <= NT - NT / 16) {
      clear_hist(s);
      if (own > rw.floor) atomicAdd(&s.hist[rw.bin(own)], 1ull);
      find_bin<false>(0.0, (u64)a.top_k, 0ull, s);
      if (s.bin >= 0) nlist = list_down_to<false>(row, V, rw, s.bin, s);
      listed = s.bin >= 0 && nlist <= s.LCAP;
    }
    clear_hist(s);
    // (tokens without weight can never be chosen: whether they count makes no difference, and masks put thousands of them
    // on one value)
    if (listed) each_of_list(s, nlist, [&](float l, int) { atomicAdd(&s.hist[rw.bin(l)], 1ull); });
    else each_of_row<NT>(row, V, rw, [&](float l, int) { if (l > rw.floor) atomicAdd(&s.hist[rw.bin(l)], 1ull); });
    const u64 target = find_bin<false>(0.0, (u64)a.top_k, 0ull, s);
    const int bin = s.bin;
    if (bin >= 0) {
      if (listed) {
        each_of_list(s, nlist, [&](float l, int i) { if (rw.bin(l) == bin) add_to_bin(s, l, i, 1ull); });
        __syncthreads();
      } else {
        nlist = list_down_to<true>(row, V, rw, bin, s);
        listed = nlist <= s.LCAP;
      }
      if (s.nbin <= s.BCAP) cut = rank_bin<false>(s.nbin, target, s);
      else refine<false>(row, V, rw, cut, bin, bin, s.base, target, s);
    }
  }

  if (listed) {
    // everything that can still be chosen is in the list
    if (a.top_p < 1.0) {
      clear_hist(s);
      each_of_list(s, nlist, [&](float l, int i) { if (kept(cut, l, i)) atomicAdd(&s.hist[rw.bin(l)], rw.weight(l)); });
      const u64 target = find_bin<true>(a.top_p, 0ull, 0ull, s);
      const int bin = s.bin;
      if (bin >= 0) {
        each_of_list(s, nlist, [&](float l, int i) { if (rw.bin(l) == bin && kept(cut, l, i)) add_to_bin(s, l, i, rw.weight(l)); });
        __syncthreads();
        if (s.nbin <= s.BCAP) cut = rank_bin<true>(s.nbin, target, s);
        else refine<true>(row, V, rw, cut, bin, bin, s.base, target, s);
      }
    }
    for (int g = threadIdx.x; g < nseg; g += NT) s.seg[g] = 0;
    __syncthreads();
    each_of_list(s, nlist, [&](float l, int i) {
      if (kept(cut, l, i)) {
        const u64 w = rw.weight(l);
        if ((double)w >= wmin) atomicAdd(&s.seg[i / SEG], w);
      }
    });
  } else {
    const bool gen = wmin > 0.0 || cut.v > -INFINITY;
    u64 front, total;
    if (a.top_p < 1.0) {
      clear_hist(s);
      if (cut.v > -INFINITY)
        each_of_row_slowly<NT>(row, V, rw, [&](float l, int i) { if (kept(cut, l, i)) atomicAdd(&s.hist[rw.bin(l)], rw.estimate(l)); });
      else
        each_of_row<NT>(row, V, rw, [&](float l, int) { atomicAdd(&s.hist[rw.bin(l)], rw.estimate(l)); });
      find_bin<true>(a.top_p, 0ull, 0ull, s);
      int lo = s.bin_lo, hi = s.bin_hi;
      if (gen) sum_segments<true, true>(row, V, rw, cut, wmin, lo, hi, s, front, total);
      else sum_segments<true, false>(row, V, rw, cut, wmin, lo, hi, s, front, total);
      u64 target = share_of(a.top_p, total);
      int n = s.nbin;
      // the bins are right when the target lies inside them (bins of -1 have nothing in front and nothing in them)
      u64 inside = 0;
      for (int t = threadIdx.x; t < (n < s.BCAP ? n : s.BCAP); t += NT) inside += s.bt[t].w;
      inside = block_sum(inside, s);
      const Cut whole = cut;
      bool found = false, ranked = false;
      if (front < target) {
        if (n > s.BCAP) {
          found = refine<true>(row, V, rw, cut, lo, hi, front, target, s);
        } else if (front + inside >= target) {
          if (threadIdx.x == 0) s.base = front;
          __syncthreads();
          cut = rank_bin<true>(n, target, s);
          found = ranked = true;
        }
      }
      if (!found) {
        // the histogram again, with the exact weights
        cut = whole;
        clear_hist(s);
        for (int g = threadIdx.x; g < nseg; g += NT) s.seg[g] = 0;
        each_of_row_slowly<NT>(row, V, rw, [&](float l, int i) {
          const u64 w = rw.weight(l);
          if (w && kept(cut, l, i)) atomicAdd(&s.hist[rw.bin(l)], w);
        });
        target = find_bin<true>(a.top_p, 0ull, 0ull, s);
        lo = hi = s.bin < 0 ? NB : s.bin;
        front = s.base;
        each_of_row_slowly<NT>(row, V, rw, [&](float l, int i) {
          const u64 w = rw.weight(l);
          if (w && rw.bin(l) < lo && kept(cut, l, i) && (double)w >= wmin) atomicAdd(&s.seg[i / SEG], w);
        });
        __syncthreads();
        if (lo < NB) refine<true>(row, V, rw, cut, lo, hi, front, target, s);
      }
      // the tokens of these bins that stay
      if (ranked) {
        for (int t = threadIdx.x; t < n; t += NT) {
          const Token k = s.bt[t];
          if (kept(cut, k.v, k.i) && (double)k.w >= wmin) atomicAdd(&s.seg[k.i / SEG], k.w);
        }
      } else if (lo < NB) {
        each_of_row_slowly<NT>(row, V, rw, [&](float l, int i) {
          const int b = rw.bin(l);
          if (b >= lo && b <= hi && kept(cut, l, i)) {
            const u64 w = rw.weight(l);
            if (w && (double)w >= wmin) atomicAdd(&s.seg[i / SEG], w);
          }
        });
      }
    } else if (gen) {
      sum_segments<false, true>(row, V, rw, cut, wmin, NB, NB, s, front, total);
    } else {
      sum_segments<false, false>(row, V, rw, cut, wmin, NB, NB, s, front, total);
    }
  }
  __syncthreads();
  if (wid != 0) return;
  u64 before, target;
  const int found = find_segment(nseg, a.u[r], before, target, s);
  const int c = found * SEG + lane * 16;
  float x[2][8];
#pragma unroll
  for (int h = 0; h < 2; ++h) load8(row, c + h * 8, V, x[h]);
  u64 w[16];
  int idx[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const float l = rw.hold(x[j / 8][j % 8]);
    idx[j] = c + j;
    w[j] = kept(cut, l, c + j) ? rw.weight(l) : 0ull;
    if ((double)w[j] < wmin) w[j] = 0ull;
  }
  choose_in_segment(w, idx, before, target, a.out + r);
}

template <int NT, int NB, typename T>
int launch(const T *logits, const FArgs &a, int64_t rows, hipStream_t s) {
  constexpr int bytes = (int)sizeof(Shared<NT, NB>);
  static std::atomic<uint64_t> attr_done{0};
  uint64_t dev_bit;
  if (ldm_attr_pending(attr_done, &dev_bit)) {
    (void)hipFuncSetAttribute((const void *)sample_filtered_k<NT, NB, T>, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    attr_done.fetch_or(dev_bit, std::memory_order_release);
  }
  hipLaunchKernelGGL((sample_filtered_k<NT, NB, T>), dim3((unsigned)rows), dim3(NT), bytes, s, logits, a);
  LDM_CHECK_LAUNCH();
  return LDM_OK;
}

// Threads and bins by what was measured (us).  A wave per row up to 1024 tokens, four up to 8192 (T = 4096, V = 1000, top_p
// 0.9: 32 against 110 for 512 threads).  With many rows, 256 threads and 2048 bins: four rows share a CU, one's barriers and
// loads under the others' arithmetic (2048 of 4096 rows, V = 30522, top_k 200 and top_p 0.95: 137 against 162 for 512
// threads and 4096 bins; V = 9000: 119 / 157); but not where a bin then outgrows its list (1000 rows, V = 126464: 590 /
// 338).  With fewer than two rows per CU, 1024 threads, for the time of one row (32 rows, V = 30522, top_p 0.9: 31 / 38).
template <typename T>
int launch_rows(const void *logits, const FArgs &a, int64_t rows, hipStream_t s) {
  const T *l = (const T *)logits;
  if (a.V <= 1024) return launch<64, 512>(l, a, rows, s);
  if (a.V <= 8192) return launch<256, 1024>(l, a, rows, s);
  if (a.V <= 65536 && rows >= 1024) return launch<256, 2048>(l, a, rows, s);
  return rows >= 512 ? launch<512, 4096>(l, a, rows, s) : launch<1024, 4096>(l, a, rows, s);
}

}  // namespace

extern "C" int ldm_sample_filtered(const void *logits, int dtype, int64_t T, int64_t V, int64_t ld, const float *u,
                                   const int64_t *ids, int64_t mask_id, double temperature, int64_t top_k, double top_p,
                                   double min_p, int64_t *out, void *stream) {
  if (T < 0 || V <= 0 || ld < V || top_k < 0) return LDM_E_BADARG;
  if (!(temperature >= 0.0) || !(top_p > 0.0) || !(min_p >= 0.0 && min_p <= 1.0)) return LDM_E_BADARG;
  if (dtype != LDM_F32 && dtype != LDM_BF16) return LDM_E_DTYPE;
  if (V > MAX_V || T > 0x7fffffff) return LDM_E_SHAPE;
  if (T == 0) return LDM_OK;
  if (!logits || !u || !out) return LDM_E_BADARG;
  const double inv = temperature > 0.0 ? 1.0 / temperature : 1.0;
  if (!(inv >= 1e-28 && inv <= 1e28)) return LDM_E_BADARG;
  FArgs a;
  a.ld = ld; a.V = (int)V; a.u = u; a.ids = ids; a.mask_id = mask_id;
  a.inv_temp = inv;
  a.top_p = top_p;
  a.min_p = min_p;
  a.top_k = temperature > 0.0 ? (int)(top_k < V ? top_k : 0) : 1;     // temperature 0: the first maximum
  if (temperature == 0.0) a.top_p = 1.0;
  // V weights of at most 2^shift add up to at most 2^62
  int bits = 0;
  while ((1ll << bits) < V) ++bits;
  a.shift = 62 - bits < 45 ? 62 - bits : 45;
  a.out = out;
  hipStream_t s = (hipStream_t)stream;
  // (a grid of 2^32 threads and more is cut off without an error: longer inputs take several launches)
  constexpr int64_t ROWS = 1 << 21;
  for (int64_t t = 0; t < T; t += ROWS) {
    const int64_t rows = T - t < ROWS ? T - t : ROWS;
    FArgs b = a;
    b.u += t;
    if (b.ids) b.ids += t;
    b.out += t;
    const int rc = dtype == LDM_F32 ? launch_rows<float>((const float *)logits + t * ld, b, rows, s)
                                    : launch_rows<bf16_t>((const bf16_t *)logits + t * ld, b, rows, s);
    if (rc != LDM_OK) return rc;
  }
  return LDM_OK;
}
