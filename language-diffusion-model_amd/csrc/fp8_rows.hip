// 8-bit rows for the inference projections: residual addition + RMSNorm with e4m3 rows out, e4m3 rows of a matrix or of
// a * silu(g), and the 128 x 128-block form for weights.  All of them are bound by memory: one pass, every element read
// once and kept in registers between the statistics and the store.
//
// Layout: a lane owns 8 consecutive columns (one 16-byte load of bf16, one 8-byte store of e4m3), so a 128-column block is
// one 16-lane DPP row and its maximum needs four register moves and no LDS.
//
// Measured (a copy of 1 GiB reaches 5.2 TB/s on the same card): addition + norm of 16384 x 4096 bf16 rows onto an fp32 stream 136
// us = 5.4 TB/s, of 15001 x 768 onto a bf16 one 17 us = 4.7 TB/s; a * silu(g) of 8191 x 5632 43 us = 5.3 TB/s; rows of 2048 x 768
// 3.3 us (a launch of next to nothing takes 3).  Odd widths lose the alignment of their rows, not the wide loads: 16384 x
// 4095 bf16 3.6 TB/s.
#include "fp8.h"

namespace {

struct NormArgs {
  const void *x; int64_t ld_x;
  const void *res; int64_t ld_res;
  const float *w;
  int64_t T; int d; float eps;
  void *out;                       // x + res as stored, [T, d] contiguous
  uint8_t *q; int64_t ld_q;
  uint8_t *scale; int64_t ld_s;
};

// G lanes per row (16: four rows per wave; 64: a wave per row; 256: a workgroup per row), NC chunks of 8 columns per lane:
// G * NC * 8 >= d.  XT: type of x; ST: type of the residual stream (res and out); RES: whether there is a residual.
// The norm is taken of the fp32 sum, before its rounding to the stream's type.
template <typename XT, typename ST, bool RES, int G, int NC>
__global__ __launch_bounds__(256) void rmsnorm_fp8_k(NormArgs a) {
  constexpr int RPB = 256 / G;
  const int lane = threadIdx.x % G;
  const int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / G;
  if (G <= 64 && row >= a.T) return;       // (a row's lanes leave together; with G = 256 every row exists)
  const XT *x = (const XT *)a.x + row * a.ld_x;
  const ST *r = RES ? (const ST *)a.res + row * a.ld_res : nullptr;
  float v[NC][8];
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int c = (lane + i * G) * 8;
    fp8_load8_tail(x, c, a.d, v[i]);
  }
  if constexpr (RES) {
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = (lane + i * G) * 8;
      float t[8];
      fp8_load8_tail(r, c, a.d, t);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] += t[j];
    }
  }
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < NC; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = fmaf(v[i][j], v[i][j], ss);
  ss = row16_sum(ss);
  if constexpr (G >= 64) {
    ss += __shfl_xor(ss, 16, 64);
    ss += __shfl_xor(ss, 32, 64);
  }
  if constexpr (G == 256) {
    __shared__ float part[4];
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = ss;
    __syncthreads();
    ss = (part[0] + part[1]) + (part[2] + part[3]);
  }
  const float rstd = 1.0f / sqrtf(ss / (float)a.d + a.eps);
  if constexpr (RES) {
    ST *o = (ST *)a.out + row * a.d;
#pragma unroll
    for (int i = 0; i < NC; ++i) fp8_store8_tail(o, (lane + i * G) * 8, a.d, v[i]);
  }
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int c = (lane + i * G) * 8;
    float w[8];
    fp8_load8_tail(a.w, c, a.d, w);
    float m = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[i][j] = v[i][j] * rstd * w[j];
      m = fmaxf(m, fp8_mag(v[i][j]));
    }
    m = row16_max(m);
    const unsigned code = fp8_scale_code(m);
    const float inv = fp8_inv_scale(code);
    if (c < a.d) {
      if (c + 8 > a.d) {      // (zeros behind the last column: 0 * rstd is NaN in a row with a NaN)
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = c + j < a.d ? v[i][j] : 0.f;
      }
      uint2 p;
      p.x = fp8_pack4(v[i][0] * inv, v[i][1] * inv, v[i][2] * inv, v[i][3] * inv);
      p.y = fp8_pack4(v[i][4] * inv, v[i][5] * inv, v[i][6] * inv, v[i][7] * inv);
      *reinterpret_cast<uint2 *>(a.q + row * a.ld_q + c) = p;
      if ((lane & 15) == 0) a.scale[row * a.ld_s + c / FP8_BLOCK] = (uint8_t)code;
    }
  }
}

struct QuantArgs {
  const void *x; int64_t ld_x;
  int64_t T; int d; int nb;        // nb: 128-column blocks per row
  uint8_t *q; int64_t ld_q;
  uint8_t *scale; int64_t ld_s;
};

// 16 lanes per 128-column block; the blocks of all rows are walked in row-major order.  SWIGLU: x is [a | g], the value is
// a * silu(g) = a * g / (1 + e^-g) (g * rcp first: for g -> -inf it is 0 * g, never inf * 0).
template <typename XT, bool SWIGLU>
__global__ __launch_bounds__(256) void quant_fp8_k(QuantArgs a) {
  const int64_t gid = (int64_t)blockIdx.x * 16 + threadIdx.x / 16;
  const int64_t row = gid / a.nb;
  if (row >= a.T) return;
  const int blk = (int)(gid - row * a.nb);
  const int c = blk * FP8_BLOCK + (threadIdx.x & 15) * 8;
  const XT *x = (const XT *)a.x + row * a.ld_x;
  float v[8];
  fp8_load8_tail(x, c, a.d, v);
  if constexpr (SWIGLU) {
    float g[8];
    fp8_load8_tail(x + a.d, c, a.d, g);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= g[j] * __builtin_amdgcn_rcpf(1.0f + __expf(-g[j]));
  }
  float m = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = fmaxf(m, fp8_mag(v[j]));
  m = row16_max(m);
  const unsigned code = fp8_scale_code(m);
  const float inv = fp8_inv_scale(code);
  if (c < a.d) {
    uint2 p;
    p.x = fp8_pack4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
    p.y = fp8_pack4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv);
    *reinterpret_cast<uint2 *>(a.q + row * a.ld_q + c) = p;
    if ((threadIdx.x & 15) == 0) a.scale[row * a.ld_s + blk] = (uint8_t)code;
  }
}

// Weights: one scale per 128 x 128 block, one workgroup per block (laid out once per weight version, not per call).
__global__ __launch_bounds__(256) void quant_fp8_block_k(const float *w, int64_t ld_w, int64_t N, int K, uint8_t *q,
                                                         int64_t ld_q, uint8_t *scale, int64_t ld_s) {
  const int64_t n0 = (int64_t)blockIdx.y * FP8_BLOCK;
  const int c = (int)blockIdx.x * FP8_BLOCK + (threadIdx.x & 15) * 8;
  const int r0 = threadIdx.x / 16;
  float v[8][8];
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t n = n0 + r0 + i * 16;
    if (n < N) {
      fp8_load8_tail(w + n * ld_w, c, K, v[i]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) m = fmaxf(m, fp8_mag(v[i][j]));
  }
  m = wave_max(m);
  __shared__ float part[4];
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = m;
  __syncthreads();
  m = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
  const unsigned code = fp8_scale_code(m);
  const float inv = fp8_inv_scale(code);
  if (threadIdx.x == 0) scale[(int64_t)blockIdx.y * ld_s + blockIdx.x] = (uint8_t)code;
  if (c >= K) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t n = n0 + r0 + i * 16;
    if (n >= N) break;
    uint2 p;
    p.x = fp8_pack4(v[i][0] * inv, v[i][1] * inv, v[i][2] * inv, v[i][3] * inv);
    p.y = fp8_pack4(v[i][4] * inv, v[i][5] * inv, v[i][6] * inv, v[i][7] * inv);
    *reinterpret_cast<uint2 *>(q + n * ld_q + c) = p;
  }
}

template <typename XT, typename ST, bool RES>
int launch_norm(const NormArgs &a, hipStream_t s) {
  const int chunks = (int)ceil_div(a.d, 8);
#define LDM_NORM(G, NC)                                                                                              \
  hipLaunchKernelGGL((rmsnorm_fp8_k<XT, ST, RES, G, NC>), dim3((unsigned)ceil_div(a.T, 256 / G)), dim3(256), 0, s, a)
  if (chunks <= 16) LDM_NORM(16, 1);
  else if (chunks <= 32) LDM_NORM(16, 2);
  else if (chunks <= 64) LDM_NORM(64, 1);
  else if (chunks <= 128) LDM_NORM(64, 2);
  else if (chunks <= 256) LDM_NORM(256, 1);
  else if (chunks <= 512) LDM_NORM(256, 2);
  else if (chunks <= 1024) LDM_NORM(256, 4);
  else LDM_NORM(256, 8);
#undef LDM_NORM
  LDM_CHECK_LAUNCH();
  return LDM_OK;
}

// Rows (or 128-column blocks of rows) of a launch: a grid of 2^32 threads and more is cut off without an error, so longer
// inputs take several launches
constexpr int64_t ROWS = 1 << 23, BLOCKS = 1 << 27;

}  // namespace

extern "C" int ldm_rmsnorm_fp8(const void *x, int x_dtype, int64_t ld_x, const void *res, int stream_dtype,
                               int64_t ld_res, const float *w, int64_t T, int64_t d, float eps, void *stream_out,
                               uint8_t *q, int64_t ld_q, uint8_t *scale, int64_t ld_s, void *stream) {
  if (T < 0 || d <= 0) return LDM_E_BADARG;
  if ((x_dtype != LDM_F32 && x_dtype != LDM_BF16) || (res && stream_dtype != LDM_F32 && stream_dtype != LDM_BF16))
    return LDM_E_DTYPE;
  if (res && x_dtype == LDM_F32 && stream_dtype == LDM_BF16) return LDM_E_DTYPE;
  if (d > 16384 || T >= (1ll << 40)) return LDM_E_SHAPE;
  if (T == 0) return LDM_OK;
  if (!x || !w || !q || !scale || (res && !stream_out)) return LDM_E_BADARG;
  if (ld_x < d || (res && ld_res < d) || ld_s < ceil_div(d, FP8_BLOCK)) return LDM_E_BADARG;
  if (ld_q % 8 || ld_q < ceil_div(d, 8) * 8 || !aligned_to(q, 8)) return LDM_E_ALIGN;
  hipStream_t s = (hipStream_t)stream;
  const int64_t xb = x_dtype == LDM_F32 ? 4 : 2, rb = stream_dtype == LDM_F32 ? 4 : 2;
  for (int64_t t = 0; t < T; t += ROWS) {
    const NormArgs a{(const char *)x + t * ld_x * xb, ld_x, res ? (const char *)res + t * ld_res * rb : nullptr, ld_res, w,
                     T - t < ROWS ? T - t : ROWS, (int)d, eps, res ? (char *)stream_out + t * d * rb : nullptr,
                     q + t * ld_q, ld_q, scale + t * ld_s, ld_s};
    int rc;
    if (!res) rc = x_dtype == LDM_F32 ? launch_norm<float, float, false>(a, s) : launch_norm<bf16_t, bf16_t, false>(a, s);
    else if (x_dtype == LDM_F32) rc = launch_norm<float, float, true>(a, s);
    else rc = stream_dtype == LDM_F32 ? launch_norm<bf16_t, float, true>(a, s) : launch_norm<bf16_t, bf16_t, true>(a, s);
    if (rc != LDM_OK) return rc;
  }
  return LDM_OK;
}

extern "C" int ldm_quant_fp8(const void *x, int dtype, int64_t ld_x, int64_t T, int64_t d, int swiglu, uint8_t *q,
                             int64_t ld_q, uint8_t *scale, int64_t ld_s, void *stream) {
  if (T < 0 || d <= 0) return LDM_E_BADARG;
  if (dtype != LDM_F32 && dtype != LDM_BF16) return LDM_E_DTYPE;
  if (d > (1 << 28)) return LDM_E_SHAPE;
  if (T == 0) return LDM_OK;
  if (!x || !q || !scale) return LDM_E_BADARG;
  const int64_t nb = ceil_div(d, FP8_BLOCK);
  if (ld_x < (swiglu ? 2 * d : d) || ld_s < nb) return LDM_E_BADARG;
  if (ld_q % 8 || ld_q < ceil_div(d, 8) * 8 || !aligned_to(q, 8)) return LDM_E_ALIGN;
  if (T >= (1ll << 40)) return LDM_E_SHAPE;
  hipStream_t s = (hipStream_t)stream;
  const int64_t most = BLOCKS / nb, xb = dtype == LDM_F32 ? 4 : 2;      // (nb <= 2^21)
  for (int64_t t = 0; t < T; t += most) {
    const int64_t rows = T - t < most ? T - t : most;
    const QuantArgs a{(const char *)x + t * ld_x * xb, ld_x, rows, (int)d, (int)nb, q + t * ld_q, ld_q, scale + t * ld_s, ld_s};
    const dim3 grid((unsigned)ceil_div(rows * nb, 16)), wg(256);
    if (dtype == LDM_F32) {
      if (swiglu) hipLaunchKernelGGL((quant_fp8_k<float, true>), grid, wg, 0, s, a);
      else hipLaunchKernelGGL((quant_fp8_k<float, false>), grid, wg, 0, s, a);
    } else {
      if (swiglu) hipLaunchKernelGGL((quant_fp8_k<bf16_t, true>), grid, wg, 0, s, a);
      else hipLaunchKernelGGL((quant_fp8_k<bf16_t, false>), grid, wg, 0, s, a);
    }
    LDM_CHECK_LAUNCH();
  }
  return LDM_OK;
}

extern "C" int ldm_quant_fp8_block(const float *w, int64_t ld_w, int64_t N, int64_t K, uint8_t *q, int64_t ld_q,
                                   uint8_t *scale, int64_t ld_s, void *stream) {
  if (N < 0 || K <= 0) return LDM_E_BADARG;
  if (N == 0) return LDM_OK;
  if (!w || !q || !scale) return LDM_E_BADARG;
  const int64_t kb = ceil_div(K, FP8_BLOCK), nb = ceil_div(N, FP8_BLOCK);
  if (ld_w < K || ld_s < kb) return LDM_E_BADARG;
  if (ld_q % 8 || ld_q < ceil_div(K, 8) * 8 || !aligned_to(q, 8)) return LDM_E_ALIGN;
  if (K > (1 << 28) || nb > 65535) return LDM_E_SHAPE;
  hipLaunchKernelGGL(quant_fp8_block_k, dim3((unsigned)kb, (unsigned)nb), dim3(256), 0, (hipStream_t)stream, w, ld_w, N,
                     (int)K, q, ld_q, scale, ld_s);
  LDM_CHECK_LAUNCH();
  return LDM_OK;
}
