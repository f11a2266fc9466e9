// Group-128 int8 quantizers.
//
//  * lm_quantize_weight_g128: the offline weight format producer
//    (convert.py:31-37): s = max(amax / 127, 1e-30), q = clamp(rne(w / s), +-127).
//  * lm_act_quant_g128: dynamic per-row activation quantization of the W8A8
//    decode path (w8a8.py:8-22): s = max(amax, 1e-10) * fl32(1/127),
//    q = rint(x / s) with IEEE division (|x / s| <= 127 by construction).
//  * lm_norm_quant_g128: rows on their way into a W8A8 product, h += x, their RMS norm and its
//    quantization in one pass.
//
// One 128-element group is handled by 32 lanes holding 4 elements each, so a
// wave quantizes two groups per iteration with fully coalesced 16-byte loads.
#include "gemv_core.hpp"

namespace lm {

__global__ __launch_bounds__(256) void quantize_weight_kernel(const float *__restrict__ w,
                                                              int8_t *__restrict__ q,
                                                              float *__restrict__ s,
                                                              int64_t ngroups) {
  const int lane = threadIdx.x & 63;
  const int l = lane & 31;
  const int64_t wave = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 6;
  const int64_t nwaves = ((int64_t)gridDim.x * blockDim.x) >> 6;
  for (int64_t g2 = wave; g2 * 2 < ngroups; g2 += nwaves) {
    const int64_t grp = g2 * 2 + (lane >> 5);
    const bool valid = grp < ngroups;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (valid) v = *reinterpret_cast<const f32x4 *>(w + grp * 128 + l * 4);
    float a = fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) a = fmaxf(a, __shfl_xor(a, o, 64));
    const float sc = fmaxf(a / 127.0f, 1e-30f);
    uint32_t packed = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float r = rintf(v[i] / sc);
      r = fminf(fmaxf(r, -127.0f), 127.0f);
      packed |= ((uint32_t)(uint8_t)(int8_t)(int)r) << (8 * i);
    }
    if (valid) {
      *reinterpret_cast<uint32_t *>(q + grp * 128 + l * 4) = packed;
      if (l == 0) s[grp] = sc;
    }
  }
}

template <typename T>
__global__ __launch_bounds__(256) void act_quant_kernel(const uint16_t *__restrict__ x,
                                                        int8_t *__restrict__ q,
                                                        float *__restrict__ s,
                                                        int64_t ngroups) {
  // A half-wave quantizes B groups per pass: all B loads are issued before
  // the first is used and the groups are computed branch-free (slots past
  // the end redo the last group and store the same bytes to it again), so a
  // pass costs one load latency.
  constexpr int B = 4;
  const int l = threadIdx.x & 31;
  const int64_t half = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int64_t nhalf = ((int64_t)gridDim.x * blockDim.x) >> 5;
  for (int64_t base = half; base < ngroups; base += nhalf * B) {
    uint2 raw[B];
#pragma unroll
    for (int u = 0; u < B; ++u) {
      const int64_t grp = min(base + u * nhalf, ngroups - 1);
      raw[u] = *reinterpret_cast<const uint2 *>(x + grp * 128 + l * 4);
    }
#pragma unroll
    for (int u = 0; u < B; ++u) {
      const int64_t grp = min(base + u * nhalf, ngroups - 1);
      quantize_group<T>(raw[u], l, q + grp * 128, s + grp);
    }
  }
}


// ------------------------------------------------------------------ norm and quantization
// h := T(h + x), n = h rsqrt(mean h^2 + eps) (1 + w), s = max(amax |n|, 1e-10) fl(1/127) of each 128,
// q = rint(n / s): n stays in fp32 until it is quantized.  A row lies in the registers of WAVES
// waves, eight values a thread and chunk, a group of 128 in 16 lanes; it is read once.  Not finite
// values leave a scale that is not.  x may be h itself: a thread's loads come before its stores.
//
// Bound by its bytes, 7 a value, 3 without x, and by a launch's start and end: 2048 rows of 2048 take
// 8.3 us from memory (29.5 MB, 3.6 TB/s; 6.4 us with the rows in the caches), without x 5.2 us; 8192
// rows 22.1 us (5.3 TB/s), without x 13.2; one row 2 us.  Divisions and a conversion for each byte
// took twice that.  A wave a row of 2048, without a barrier, took 8.1 us instead of 7.5.
template <typename T, int WAVES, int CHUNKS, bool ADD>
__global__ __launch_bounds__(256) void norm_quant_kernel(uint16_t *h, const uint16_t *x,
                                                         const float *__restrict__ w,
                                                         int8_t *__restrict__ q,
                                                         float *__restrict__ s, int64_t rows, int n,
                                                         float eps) {
  constexpr int THREADS = WAVES * 64;
  __shared__ float sums[4];
  const int tid = threadIdx.x % THREADS;
  const int64_t row = (int64_t)blockIdx.x * (4 / WAVES) + threadIdx.x / THREADS;
  if (WAVES == 1 && row >= rows) return;  // with more waves a workgroup has one row
  const int64_t at = row * n;
  float v[CHUNKS][8], g[CHUNKS][8];
  u32x4 a[CHUNKS], b[CHUNKS];
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int i = min((c * THREADS + tid) * 8, n - 8);  // again the last, where there is no more
    a[c] = ldg16(h + at + i);
    if constexpr (ADD) b[c] = ldg16(x + at + i);
    if (w) {
      *reinterpret_cast<f32x4 *>(g[c]) = *reinterpret_cast<const f32x4 *>(w + i);
      *reinterpret_cast<f32x4 *>(g[c] + 4) = *reinterpret_cast<const f32x4 *>(w + i + 4);
    }
  }
  float ss = 0.0f;
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int i = (c * THREADS + tid) * 8;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (ADD)
        a[c][j] = T::pack2(T::to_f32(a[c][j] & 0xFFFFu) + T::to_f32(b[c][j] & 0xFFFFu),
                           T::to_f32(a[c][j] >> 16) + T::to_f32(b[c][j] >> 16));
      v[c][2 * j] = T::to_f32(a[c][j] & 0xFFFFu);
      v[c][2 * j + 1] = T::to_f32(a[c][j] >> 16);
    }
    if (i < n) {
      if constexpr (ADD) *reinterpret_cast<u32x4 *>(h + at + i) = a[c];
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = __builtin_fmaf(v[c][j], v[c][j], ss);
    }
  }
  ss = wave_sum_f32(ss);
  if constexpr (WAVES > 1) {
    if ((tid & 63) == 0) sums[tid >> 6] = ss;
    __syncthreads();
    ss = (sums[0] + sums[1]) + (sums[2] + sums[3]);
  }
  const float scale = 1.0f / sqrtf(ss / (float)n + eps);
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int i = (c * THREADS + tid) * 8;
    if (i >= n) break;  // 16 lanes at a time
    float most = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[c][j] *= scale;
      if (w) v[c][j] *= 1.0f + g[c][j];
      most = __builtin_elementwise_maximum(most, fabsf(v[c][j]));  // NaN above all
    }
    uint32_t bits = __float_as_uint(most);
    bits = max(bits, dpp_u32<0xB1>(bits));
    bits = max(bits, dpp_u32<0x4E>(bits));
    bits = max(bits, dpp_u32<0x141>(bits));
    bits = max(bits, dpp_u32<0x140>(bits));
    const float amax = __uint_as_float(max(bits, __float_as_uint(1e-10f)));
    const float group = amax * (1.0f / 127.0f), inverse = 1.0f / group;
    // The quotient, at most 127 and half a step, plus 1.5 * 2^23 is rint of it in the low byte.
    uint32_t b[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      b[j] = __float_as_uint(quant_div(v[c][j], group, inverse) + 12582912.0f);
    auto bytes = [&](int j) {
      return __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[j + 3], b[j + 2], 0x0C0C0400u),
                                   __builtin_amdgcn_perm(b[j + 1], b[j], 0x0C0C0400u), 0x05040100u);
    };
    *reinterpret_cast<uint2 *>(q + at + i) = uint2{bytes(0), bytes(4)};
    if ((tid & 15) == 0) s[(at + i) / 128] = group;
  }
}

template <typename T, bool ADD>
static int launch_norm_quant(void *h, const void *x, const float *w, int8_t *q, float *s,
                             int64_t rows, int64_t n, float eps, hipStream_t st) {
  uint16_t *hp = static_cast<uint16_t *>(h);
  const uint16_t *xp = static_cast<const uint16_t *>(x);
  const unsigned grid = (unsigned)rows;
  if (n <= 512)  // a wave a row, longer ones four
    norm_quant_kernel<T, 1, 1, ADD><<<(grid + 3) / 4, 256, 0, st>>>(hp, xp, w, q, s, rows, (int)n,
                                                                     eps);
  else if (n <= 2048)
    norm_quant_kernel<T, 4, 1, ADD><<<grid, 256, 0, st>>>(hp, xp, w, q, s, rows, (int)n, eps);
  else if (n <= 4096)
    norm_quant_kernel<T, 4, 2, ADD><<<grid, 256, 0, st>>>(hp, xp, w, q, s, rows, (int)n, eps);
  else if (n <= 8192)
    norm_quant_kernel<T, 4, 4, ADD><<<grid, 256, 0, st>>>(hp, xp, w, q, s, rows, (int)n, eps);
  else
    norm_quant_kernel<T, 4, 8, ADD><<<grid, 256, 0, st>>>(hp, xp, w, q, s, rows, (int)n, eps);
  return check_launch("norm_quant_kernel");
}

static unsigned quant_grid(int64_t ngroups) {
  int64_t waves = (ngroups + 1) / 2;
  int64_t blocks = (waves + 3) / 4;
  if (blocks > 4096) blocks = 4096;
  return (unsigned)(blocks < 1 ? 1 : blocks);
}

// act_quant_kernel: one half-wave per 4 groups (8 half-waves per block).
static unsigned act_quant_grid(int64_t ngroups) {
  int64_t blocks = (ngroups + 31) / 32;
  if (blocks > 4096) blocks = 4096;
  return (unsigned)(blocks < 1 ? 1 : blocks);
}

}  // namespace lm

using namespace lm;

extern "C" int lm_quantize_weight_g128(const float *w, int8_t *q, float *s, int64_t rows,
                                       int64_t k, void *stream) {
  LM_REQUIRE(rows >= 0 && k > 0 && k % 128 == 0, LM_EINVAL, "Invalid INT8 group geometry");
  LM_REQUIRE(rows == 0 || (w && q && s), LM_EINVAL, "null pointer");
  const int64_t ngroups = rows * (k / 128);
  if (ngroups == 0) return LM_OK;
  quantize_weight_kernel<<<quant_grid(ngroups), 256, 0, as_stream(stream)>>>(w, q, s, ngroups);
  return check_launch("quantize_weight_kernel");
}

// The 16-row tile layout of an int8 bank (lm_w8_tile_rows): one wave per
// 1 KB block (16 rows x 64 K of one expert); lane 16 p + r copies piece p
// (16 bytes) of row r to byte 16 (16 p + r) of the block.  The fp16 format
// (LM_TILES_F16) also biases each byte to u = q + 128 and stores the bytes of
// every dword in the order k = 0, 2, 1, 3, which the GEMM's fp16 conversion
// takes apart with one mask and one byte permute.
__global__ __launch_bounds__(256) void tile_rows_kernel(const int8_t *__restrict__ q,
                                                        int8_t *__restrict__ tiles, int64_t blocks,
                                                        int64_t nb, int64_t kb, int64_t k,
                                                        int64_t es, int fmt) {
  const int64_t blk = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (blk >= blocks) return;
  const int lane = threadIdx.x & 63, p = lane >> 4, r = lane & 15;
  const int64_t e = blk / (nb * kb), rem = blk - e * nb * kb;
  const int64_t b = rem / kb, s = rem - b * kb;
  u32x4 v = ldg16(q + e * es + (16 * b + r) * k + 64 * s + 16 * p);
  if (fmt == LM_TILES_F16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t u = v[i] ^ 0x80808080u;
      v[i] = (u & 0xFF0000FFu) | ((u >> 8) & 0x0000FF00u) | ((u << 8) & 0x00FF0000u);
    }
  }
  *reinterpret_cast<u32x4 *>(tiles + e * es + (b * kb + s) * 1024 + lane * 16) = v;
}

extern "C" int lm_w8_tile_rows(const int8_t *q, int64_t experts, int64_t n, int64_t k,
                               int64_t expert_stride, int8_t *tiles, int format, void *stream) {
  LM_REQUIRE(experts >= 0 && n > 0 && k > 0 && n % 16 == 0 && k % 64 == 0, LM_EINVAL,
             "the tile layout needs n % 16 == 0 and k % 64 == 0");
  LM_REQUIRE(expert_stride >= n * k, LM_EINVAL, "expert stride smaller than n * k");
  LM_REQUIRE(format == LM_TILES_PLAIN || format == LM_TILES_F16, LM_EINVAL,
             "unknown tile format");
  LM_REQUIRE(experts == 0 || (q && tiles), LM_EINVAL, "null pointer");
  const int64_t nb = n / 16, kb = k / 64, blocks = experts * nb * kb;
  if (blocks == 0) return LM_OK;
  LM_REQUIRE((blocks + 3) / 4 < (int64_t(1) << 31), LM_EINVAL, "bank too large for one launch");
  tile_rows_kernel<<<(unsigned)((blocks + 3) / 4), 256, 0, as_stream(stream)>>>(
      q, tiles, blocks, nb, kb, k, expert_stride, format);
  return check_launch("tile_rows_kernel");
}

extern "C" int lm_act_quant_g128(const void *x, int x_dtype, int8_t *q, float *s, int64_t rows,
                                 int64_t k, void *stream) {
  LM_REQUIRE(rows >= 0 && k > 0 && k % 128 == 0, LM_EINVAL,
             "Expected CUDA rows with K divisible by 128");
  LM_REQUIRE(x_dtype == LM_BF16 || x_dtype == LM_FP16, LM_EINVAL,
             "Expected CUDA rows with K divisible by 128");
  LM_REQUIRE(rows == 0 || (x && q && s), LM_EINVAL, "null pointer");
  const int64_t ngroups = rows * (k / 128);
  if (ngroups == 0) return LM_OK;
  const uint16_t *xp = static_cast<const uint16_t *>(x);
  if (x_dtype == LM_BF16)
    act_quant_kernel<BF16><<<act_quant_grid(ngroups), 256, 0, as_stream(stream)>>>(xp, q, s, ngroups);
  else
    act_quant_kernel<FP16><<<act_quant_grid(ngroups), 256, 0, as_stream(stream)>>>(xp, q, s, ngroups);
  return check_launch("act_quant_kernel");
}

extern "C" int lm_norm_quant_g128(void *h, const void *x, const float *w, int8_t *q, float *s,
                                  int64_t rows, int64_t n, float eps, int dtype, void *stream) {
  LM_REQUIRE(rows >= 0 && rows < (1LL << 24), LM_EINVAL, "invalid number of rows");
  LM_REQUIRE(n >= 128 && n % 128 == 0 && n <= 16384, LM_EINVAL,
             "Expected rows of 128 to 16384 values, a multiple of 128");
  LM_REQUIRE(dtype == LM_BF16 || dtype == LM_FP16, LM_EINVAL,
             "Expected CUDA rows with K divisible by 128");
  if (rows == 0) return LM_OK;
  LM_REQUIRE(h && q && s, LM_EINVAL, "null pointer");
  LM_REQUIRE(((reinterpret_cast<uintptr_t>(h) | reinterpret_cast<uintptr_t>(x) |
               reinterpret_cast<uintptr_t>(w)) & 15) == 0 &&
                 (reinterpret_cast<uintptr_t>(q) & 7) == 0,
             LM_EINVAL, "rows must be 16-byte aligned");
  hipStream_t st = as_stream(stream);
  if (dtype == LM_BF16)
    return x ? launch_norm_quant<BF16, true>(h, x, w, q, s, rows, n, eps, st)
             : launch_norm_quant<BF16, false>(h, x, w, q, s, rows, n, eps, st);
  return x ? launch_norm_quant<FP16, true>(h, x, w, q, s, rows, n, eps, st)
           : launch_norm_quant<FP16, false>(h, x, w, q, s, rows, n, eps, st);
}
