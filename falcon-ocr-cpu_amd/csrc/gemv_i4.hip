// Decode GEMV (1..=8 rows) of 4-bit codes with one FP32 scale per 32, 64 or 128
// input columns, and the kernels around that storage (linear4.hpp): upload,
// dequantization, unpacking for the prefill kernels.
//
//   out[r][n] = epilogue(sum_k x'[r][k] c[n][k] s[n][k / group])
//
// with x' the input row, times a row scale or RMS-normalized if asked.
//
// Mathematics. Each 64 columns of a row of x' are written as integers
// x' = i 2^(e - 22), |i| <= 2^22, 2^e above their largest magnitude, and i as
// three signed bytes, i = d0 + 256 d1 + 65536 d2. The INT8 matrix instruction
// then forms the exact sums of 16 channels' codes times the three bytes of up to
// five rows (eight in two instructions) over the 64 columns: operands are
// the codes as the tile holds them (no conversion) and the bytes, one
// column of the product per (row, byte). A sum is at most 64 * 128 * 128 = 2^20, so
// its FP32 value is exact, and the only roundings are x' to 2^-23 of its
// group's largest magnitude (FP32's own half step there), and the FP32 products
// and sums of the group results. A row that holds an infinity or NaN is computed
// by FP32 multiply-adds instead, column after column.
#include <type_traits>

#include "linear4.hpp"

namespace focr {
namespace {

using namespace linear4;

typedef int v4i __attribute__((ext_vector_type(4)));

constexpr int kWaves = 8;
constexpr size_t kLdsBytes = 160 * 1024;

struct Args {
  const uint4 *tiles;
  const float *scales;
  const int32_t *exc_cols;
  const float *exc_vals;
  int n_exc;
  const float *x, *row_scale;
  float *out;
  int m, n, k, group, steps, tiles_total, rms, epilogue;
};

// The largest of the 16 lanes of a DPP row, in every one of them.
__device__ __forceinline__ uint32_t row_max16(uint32_t v) {
  auto other = [](uint32_t x, auto ctrl) {
    return static_cast<uint32_t>(
        __builtin_amdgcn_update_dpp(0, static_cast<int>(x), decltype(ctrl)::value, 0xf, 0xf, false));
  };
  uint32_t o = other(v, std::integral_constant<int, 0x128>());
  v = o > v ? o : v;
  o = other(v, std::integral_constant<int, 0x124>());
  v = o > v ? o : v;
  o = other(v, std::integral_constant<int, 0x122>());
  v = o > v ? o : v;
  o = other(v, std::integral_constant<int, 0x121>());
  return o > v ? o : v;
}

// The value N lanes up in the 16 lanes of a DPP row, cyclically.
template <int N>
__device__ __forceinline__ float row_up(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x120 + 16 - N, 0xf, 0xf, false));
}

// NB: 16-column blocks of the product: one for up to 5 rows (column 5 d + r holds
// byte d of row r), two for up to 8 (column 8 d + r). SK: waves that share a tile's
// steps. G: columns per scale.
template <int NB, int SK, int G>
__global__ __launch_bounds__(64 * kWaves) void gemv4_kernel(Args a) {
  constexpr int CW = 16 * NB, RS = NB == 1 ? 5 : 8;
  constexpr int NS = kStep / G;      // scales of a channel per step
  constexpr int SLOTS = kWaves / SK;  // tiles a workgroup has at once
  constexpr int WINDOW = 4;          // steps of a wave in flight
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int groups = 2 * a.steps;
  char *digits = lds;                                                    // [groups][4][CW][16 B]
  float *factors = reinterpret_cast<float *>(lds + static_cast<size_t>(groups) * 64 * CW);  // [groups][CW]
  float *red = factors + groups * CW;                                    // [kWaves][8][16]
  float *row_factor = red + kWaves * 8 * 16;                             // [8]
  uint32_t *bad = reinterpret_cast<uint32_t *>(row_factor + 8);          // [8]
  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, kg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int slot = wave / SK, part = wave % SK;
  const int M = a.m, k = a.k, steps = a.steps;

  // The wave's work: steps part, part + SK, ... (J of them, past the last one
  // masked) of tiles first, first + stride, ...
  const int J = (steps + SK - 1) / SK;
  const int stride = gridDim.x * SLOTS;
  const int rounds = (a.tiles_total + stride - 1) / stride;
  const int total = rounds * J;
  uint4 codes[WINDOW];
  float4 scales[WINDOW][NS];
  int load_round = 0, load_j = 0;
  auto load = [&](uint4 &c, float4(&s)[NS]) {
    int tile = slot + SLOTS * blockIdx.x + load_round * stride;
    tile = tile < a.tiles_total ? tile : a.tiles_total - 1;
    int step = part + SK * load_j;
    step = step < steps ? step : steps - 1;
    const size_t at = static_cast<size_t>(tile) * steps + step;
    c = a.tiles[at * 64 + lane];
#pragma unroll
    for (int i = 0; i < NS; i++) s[i] = *reinterpret_cast<const float4 *>(a.scales + (at * NS + i) * kTile + 4 * kg);
    if (++load_j == J) {
      load_j = 0;
      load_round++;
    }
  };
#pragma unroll
  for (int i = 0; i < WINDOW; i++) load(codes[i], scales[i]);

  // x' as bytes, in the order the matrix instruction reads them.
  const bool vec = k % 4 == 0 && (reinterpret_cast<uintptr_t>(a.x) & 15) == 0;
  auto load_x = [&](int r, int col) {
    const float *row = a.x + static_cast<size_t>(r) * k;
    if (vec) return col < k ? *reinterpret_cast<const float4 *>(row + col) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    return make_float4(col < k ? row[col] : 0.0f, col + 1 < k ? row[col + 1] : 0.0f, col + 2 < k ? row[col + 2] : 0.0f,
                       col + 3 < k ? row[col + 3] : 0.0f);
  };
  if (tid < 8) {
    bad[tid] = 0;
    row_factor[tid] = a.row_scale && tid < M ? a.row_scale[tid] : 1.0f;
  }
  if (a.rms) {
    for (int r = wave; r < M; r += kWaves) {
      float sum = 0.0f;
      for (int col = 4 * lane; col < k; col += 256) {
        const float4 v = load_x(r, col);
        sum = fmaf_(v.x, v.x, sum);
        sum = fmaf_(v.y, v.y, sum);
        sum = fmaf_(v.z, v.z, sum);
        sum = fmaf_(v.w, v.w, sum);
      }
#pragma unroll
      for (int mask = 32; mask >= 1; mask /= 2) sum = sum + __shfl_xor(sum, mask);
      if (lane == 0)
        red[r] = __fdiv_rn(1.0f, __builtin_sqrtf(__fdiv_rn(sum, static_cast<float>(k)) + 1.1920929e-7f));
    }
  }
  __syncthreads();
  if (a.rms && tid < M) row_factor[tid] = red[tid];
  __syncthreads();
  const bool scaled = a.rms || a.row_scale;
  for (int u = wave * 4 + kg; u < M * groups; u += kWaves * 4) {
    const int r = u / groups, g = u - r * groups;
    float4 v = load_x(r, 64 * g + 4 * l16);
    if (scaled) {
      const float f = row_factor[r];
      v = make_float4(v.x * f, v.y * f, v.z * f, v.w * f);
    }
    uint32_t big = __float_as_uint(v.x) & 0x7fffffffu;
    const uint32_t by = __float_as_uint(v.y) & 0x7fffffffu, bz = __float_as_uint(v.z) & 0x7fffffffu,
                   bw = __float_as_uint(v.w) & 0x7fffffffu;
    big = by > big ? by : big;
    big = bz > big ? bz : big;
    big = bw > big ? bw : big;
    big = row_max16(big);
    if (big >= 0x7f800000u) bad[r] = 1;
    int e = big >= 0x7f800000u || big == 0 ? 0 : __builtin_amdgcn_frexp_expf(__uint_as_float(big));
    e = e < -96 ? -96 : e;
    // 1.5 2^23 + i holds the integer i in its low bits; adding 128 to each
    // byte of i and inverting their top bits leaves signed bytes whose weighted
    // sum is i.
    auto bytes = [&](float f) {
      const float t = __builtin_ldexpf(f, 22 - e) + 12582912.0f;
      return (__float_as_uint(t) + (0x00808080u - 0x4b400000u)) ^ 0x00808080u;
    };
    const uint32_t w0 = bytes(v.x), w1 = bytes(v.y), w2 = bytes(v.z), w3 = bytes(v.w);
    const uint32_t a01 = __builtin_amdgcn_perm(w1, w0, 0x05010400u), a23 = __builtin_amdgcn_perm(w3, w2, 0x05010400u);
    const uint32_t b01 = __builtin_amdgcn_perm(w1, w0, 0x0c0c0602u), b23 = __builtin_amdgcn_perm(w3, w2, 0x0c0c0602u);
    const uint32_t d[3] = {__builtin_amdgcn_perm(a23, a01, 0x05040100u), __builtin_amdgcn_perm(a23, a01, 0x07060302u),
                           __builtin_amdgcn_perm(b23, b01, 0x05040100u)};
    char *to = digits + (static_cast<size_t>(g * 4 + l16 / 4) * CW + r) * 16 + 4 * (l16 % 4);
#pragma unroll
    for (int i = 0; i < 3; i++) *reinterpret_cast<uint32_t *>(to + i * RS * 16) = d[i];
    if (l16 < 3) factors[g * CW + l16 * RS + r] = __builtin_ldexpf(1.0f, e - 26 + 8 * l16);
  }
  __syncthreads();

  float acc[NB][4];
#pragma unroll
  for (int b = 0; b < NB; b++)
#pragma unroll
    for (int i = 0; i < 4; i++) acc[b][i] = 0.0f;
  auto consume = [&](const uint4 &c, const float4(&s)[NS], int step) {
    const uint32_t word[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
    for (int half = 0; half < 2; half++) {
      const int g = 2 * step + half;
      v4i A;
#pragma unroll
      for (int w = 0; w < 2; w++) {
        A[2 * w] = static_cast<int>((word[2 * half + w] << 4) & 0xf0f0f0f0u);
        A[2 * w + 1] = static_cast<int>(word[2 * half + w] & 0xf0f0f0f0u);
      }
#pragma unroll
      for (int b = 0; b < NB; b++) {
        const v4i B = *reinterpret_cast<const v4i *>(digits + (static_cast<size_t>(g * 4 + kg) * CW + 16 * b + l16) * 16);
        const float f = factors[g * CW + 16 * b + l16];
        const v4i zero = {0, 0, 0, 0};
        auto add = [&](const v4i &sum, const float4 &sc) {
          const float q[4] = {sc.x, sc.y, sc.z, sc.w};
#pragma unroll
          for (int i = 0; i < 4; i++) acc[b][i] = fmaf_(static_cast<float>(sum[i]) * q[i], f, acc[b][i]);
        };
        if constexpr (G >= 64) {
          add(__builtin_amdgcn_mfma_i32_16x16x64_i8(A, B, zero, 0, 0, 0), s[G == 64 ? half : 0]);
        } else {
          // Two scales in the 64 columns: lanes of the other 32 give zeros.
          const v4i lo = kg < 2 ? B : zero, hi = kg < 2 ? zero : B;
          add(__builtin_amdgcn_mfma_i32_16x16x64_i8(A, lo, zero, 0, 0, 0), s[2 * half]);
          add(__builtin_amdgcn_mfma_i32_16x16x64_i8(A, hi, zero, 0, 0, 0), s[2 * half + 1]);
        }
      }
    }
  };

  // The rows of a finished tile: lane l16 = row, channels 4 kg .. + 3.
  auto finish = [&](int round) {
    const int tile = slot + SLOTS * blockIdx.x + round * stride;
    float total[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if constexpr (NB == 1)
        total[i] = (acc[0][i] + row_up<5>(acc[0][i])) + row_up<10>(acc[0][i]);
      else
        total[i] = (acc[0][i] + row_up<8>(acc[0][i])) + acc[1][i];
#pragma unroll
      for (int b = 0; b < NB; b++) acc[b][i] = 0.0f;
    }
    if constexpr (SK > 1) {
      if (part > 0 && l16 < 8)
        *reinterpret_cast<float4 *>(red + (wave * 8 + l16) * 16 + 4 * kg) = make_float4(total[0], total[1], total[2], total[3]);
      __syncthreads();
      if (part == 0 && l16 < 8) {
#pragma unroll
        for (int p = 1; p < SK; p++) {
          const float4 v = *reinterpret_cast<const float4 *>(red + ((wave + p) * 8 + l16) * 16 + 4 * kg);
          total[0] += v.x;
          total[1] += v.y;
          total[2] += v.z;
          total[3] += v.w;
        }
      }
      __syncthreads();
      if (part > 0) return;
    }
    const int r = l16, ch = tile * kTile + 4 * kg;
    if (r >= M || tile >= a.tiles_total || ch >= a.n) return;
    const float *row = a.x + static_cast<size_t>(r) * k;
    const float rf = row_factor[r];
    auto x_at = [&](int col) { return scaled ? row[col] * rf : row[col]; };
    if (bad[r]) {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        total[i] = 0.0f;
        if (ch + i >= a.n) continue;
        for (int col = 0; col < k; col++) {
          const float w = static_cast<float>(code_at(reinterpret_cast<const uint8_t *>(a.tiles), steps, ch + i, col)) *
                          scale_at(a.scales, steps, G, ch + i, col);
          total[i] = fmaf_(x_at(col), w, total[i]);
        }
      }
    }
    for (int e = 0; e < a.n_exc; e++) {
      const float v = x_at(a.exc_cols[e]);
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (ch + i < a.n) total[i] = fmaf_(v, a.exc_vals[static_cast<size_t>(ch + i) * a.n_exc + e], total[i]);
    }
    if (a.epilogue == FOCR_EPI_GLU) {
      float *out = a.out + static_cast<size_t>(r) * (a.n / 2) + ch / 2;
      out[0] = squared_relu_glu(total[0], total[1]);
      if (ch + 2 < a.n) out[1] = squared_relu_glu(total[2], total[3]);
      return;
    }
    float *out = a.out + static_cast<size_t>(r) * a.n + ch;
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (ch + i < a.n) out[i] = a.epilogue == FOCR_EPI_ADD ? out[i] + total[i] : total[i];
  };

  int round = 0, j = 0;
  for (int base = 0; base < total; base += WINDOW) {
#pragma unroll
    for (int i = 0; i < WINDOW; i++) {
      if (base + i < total) {
        const int step = part + SK * j;
        if (step < steps) consume(codes[i], scales[i], step);
        if (++j == J) {
          finish(round);
          j = 0;
          round++;
        }
        if (base + i + WINDOW < total) load(codes[i], scales[i]);
      }
    }
  }
}

size_t lds_bytes(int nb, size_t steps) {
  const size_t cw = 16 * nb;
  return 2 * steps * (64 * cw + 4 * cw) + kWaves * 8 * 16 * 4 + 8 * 4 + 8 * 4;
}

template <int NB, int SK, int G>
int launch_one(Ctx *ctx, const Args &a, int blocks, size_t lds) {
  // Above 64 KB the attribute has to allow it; once per device and kernel.
  static bool allowed[64] = {};
  if (lds > 64 * 1024 && !(ctx->device < 64 && allowed[ctx->device])) {
    FOCR_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void *>(gemv4_kernel<NB, SK, G>),
                                       hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kLdsBytes)));
    if (ctx->device < 64) allowed[ctx->device] = true;
  }
  hipLaunchKernelGGL((gemv4_kernel<NB, SK, G>), dim3(blocks), dim3(64 * kWaves), lds, ctx->stream, a);
  FOCR_HIP_CHECK(hipGetLastError());
  return FOCR_OK;
}

template <int NB, int G>
int launch_parts(Ctx *ctx, const Args &a, size_t lds) {
  // Waves per tile: enough to give each SIMD two.
  const int sk = a.tiles_total >= 2048 ? 1 : a.tiles_total >= 512 ? 4 : 8;
  const int slots = kWaves / sk;
  const int want = (a.tiles_total + slots - 1) / slots;
  const int blocks = want < 512 ? want : 512;
  switch (sk) {
    case 1: return launch_one<NB, 1, G>(ctx, a, blocks, lds);
    case 4: return launch_one<NB, 4, G>(ctx, a, blocks, lds);
    default: return launch_one<NB, 8, G>(ctx, a, blocks, lds);
  }
}

template <int NB>
int launch_group(Ctx *ctx, const Args &a, size_t lds) {
  switch (a.group) {
    case 32: return launch_parts<NB, 32>(ctx, a, lds);
    case 64: return launch_parts<NB, 64>(ctx, a, lds);
    default: return launch_parts<NB, 128>(ctx, a, lds);
  }
}

// ---- storage -------------------------------------------------------------------
// Row-major codes, a byte each, into tiles; bit 0 of `faults`: a code outside
// -8..7, bit 1: a nonzero code whose scale is zero.
__global__ __launch_bounds__(256) void pack_kernel(const int8_t *__restrict__ codes, const float *__restrict__ scales,
                                                   int n, int k, int group, int groups, int steps, size_t chunks,
                                                   uint4 *__restrict__ tiles, uint32_t *__restrict__ faults) {
  for (size_t at = blockIdx.x * static_cast<size_t>(256) + threadIdx.x; at < chunks;
       at += static_cast<size_t>(gridDim.x) * 256) {
    const int lane = static_cast<int>(at % 64), step = static_cast<int>(at / 64 % steps);
    const int row = static_cast<int>(at / 64 / steps) * kTile + lane % 16;
    uint32_t word[4] = {0, 0, 0, 0}, fault = 0;
    if (row < n)
      for (int half = 0; half < 2; half++)
        for (int j = 0; j < 16; j++) {
          const int col = step * kStep + half * 64 + lane / 16 * 16 + j;
          if (col >= k) break;
          const int c = codes[static_cast<size_t>(row) * k + col];
          if (c < -8 || c > 7) fault |= 1;
          if (c != 0 && scales[static_cast<size_t>(row) * groups + col / group] == 0.0f) fault |= 2;
          word[2 * half + j / 8] |= static_cast<uint32_t>(c & 15) << (8 * (j % 4) + (j % 8 >= 4 ? 4 : 0));
        }
    tiles[at] = make_uint4(word[0], word[1], word[2], word[3]);
    if (fault) atomicOr(faults, fault);
  }
}

__global__ __launch_bounds__(256) void pack_scales_kernel(const float *__restrict__ scales, int n, int group, int groups,
                                                          int per, size_t count, float *__restrict__ tiled) {
  // [tile][step][per][16]; per = groups of a step.
  const int steps = (groups + per - 1) / per;
  for (size_t at = blockIdx.x * static_cast<size_t>(256) + threadIdx.x; at < count;
       at += static_cast<size_t>(gridDim.x) * 256) {
    const size_t row = at / kTile / per / steps * kTile + at % kTile;
    const size_t g = at / kTile / per % steps * per + at / kTile % per;
    tiled[at] = row < static_cast<size_t>(n) && g < static_cast<size_t>(groups) ? scales[row * groups + g] : 0.0f;
  }
}

__global__ __launch_bounds__(256) void dequantize4bit_kernel(const uint8_t *__restrict__ tiles,
                                                             const float *__restrict__ scales,
                                                             const int16_t *__restrict__ exc_index,
                                                             const float *__restrict__ exc_vals, int n_exc, size_t n,
                                                             size_t k, size_t group, size_t steps,
                                                             float *__restrict__ out) {
  for (size_t i = blockIdx.x * static_cast<size_t>(256) + threadIdx.x; i < n * k;
       i += static_cast<size_t>(gridDim.x) * 256) {
    const size_t row = i / k, col = i % k;
    float w = static_cast<float>(code_at(tiles, steps, row, col)) * scale_at(scales, steps, group, row, col);
    if (exc_index && exc_index[col] >= 0) w = exc_vals[row * n_exc + exc_index[col]];
    out[i] = w;
  }
}

// The codes as bytes: row-major, or (PANEL) in the INT16 panels' order
// [64-column group][16-channel block][lane][16].
template <bool PANEL>
__global__ __launch_bounds__(256) void unpack_kernel(const uint8_t *__restrict__ tiles, size_t n, size_t k, size_t steps,
                                                     int8_t *__restrict__ out) {
  for (size_t i = blockIdx.x * static_cast<size_t>(256) + threadIdx.x; i < n * k;
       i += static_cast<size_t>(gridDim.x) * 256) {
    size_t row = i / k, col = i % k;
    if constexpr (PANEL) {
      const size_t lane = i / 16 % 64, blocks = n / 16, block = i / 1024 % blocks, g = i / 1024 / blocks;
      row = block * 16 + lane % 16;
      col = g * 64 + lane / 16 * 16 + i % 16;
    }
    out[i] = static_cast<int8_t>(code_at(tiles, steps, row, col));
  }
}

// The INT16 panels' per-(group, channel) sums of codes times 128, and scales.
__global__ __launch_bounds__(256) void panel_sums_kernel(const uint8_t *__restrict__ tiles, const float *__restrict__ scales,
                                                         size_t n, size_t groups, size_t steps,
                                                         int32_t *__restrict__ sums, float *__restrict__ group_scales) {
  const size_t i = blockIdx.x * static_cast<size_t>(256) + threadIdx.x;
  if (i >= n * groups) return;
  const size_t g = i / n, row = i % n;
  int32_t s = 0;
  for (int j = 0; j < 64; j++) s += code_at(tiles, steps, row, g * 64 + j);
  sums[i] = 128 * s;
  group_scales[i] = scale_at(scales, steps, 64, row, g * 64);
}

unsigned blocks_for(size_t count) {
  const size_t want = (count + 255) / 256;
  return static_cast<unsigned>(want < 65536 ? (want ? want : 1) : 65536);
}

}  // namespace

int launch_gemv4(Ctx *ctx, const Linear *lin, const float *x, size_t rows, const float *row_scale, int epilogue,
                 float *out, bool rms_norm) {
  FOCR_HIP_CHECK(hipSetDevice(ctx->device));
  const size_t steps = steps_of(lin->k), width = epilogue == FOCR_EPI_GLU ? lin->n / 2 : lin->n;
  FOCR_REQUIRE(lds_bytes(1, steps) <= kLdsBytes, FOCR_E_SHAPE, "GEMV: in_dim too large for the rows of x in LDS");
  const size_t chunk = lds_bytes(2, steps) <= kLdsBytes ? 8 : 5;
  for (size_t r0 = 0; r0 < rows; r0 += chunk) {
    const size_t m = rows - r0 < chunk ? rows - r0 : chunk;
    Args a = {};
    a.tiles = static_cast<const uint4 *>(lin->gemv_codes);
    a.scales = lin->gemv_scales;
    a.exc_cols = lin->exc_cols;
    a.exc_vals = lin->exc_vals;
    a.n_exc = static_cast<int>(lin->n_exc);
    a.x = x + r0 * lin->k;
    a.row_scale = row_scale ? row_scale + r0 : nullptr;
    a.out = out + r0 * width;
    a.m = static_cast<int>(m);
    a.n = static_cast<int>(lin->n);
    a.k = static_cast<int>(lin->k);
    a.group = static_cast<int>(lin->group);
    a.steps = static_cast<int>(steps);
    a.tiles_total = static_cast<int>(lin->gemv_tiles);
    a.rms = rms_norm ? 1 : 0;
    a.epilogue = epilogue;
    const int nb = m <= 5 ? 1 : 2;
    const int rc = nb == 1 ? launch_group<1>(ctx, a, lds_bytes(1, steps)) : launch_group<2>(ctx, a, lds_bytes(2, steps));
    if (rc != FOCR_OK) return rc;
  }
  return FOCR_OK;
}

int pack_linear4(Ctx *ctx, Linear *lin, const int8_t *codes, size_t *total) {
  const size_t n = lin->n, k = lin->k, steps = steps_of(k), tiles = tiles_of(n), per = kStep / lin->group;
  lin->gemv_tiles = tiles;
  lin->gemv_steps = steps;
  const size_t chunks = tiles * steps * 64, scale_count = tiles * steps * per * kTile;
  const bool panels = lin->group == 64 && n % 32 == 0 && k % 64 == 0;
  int8_t *raw = nullptr;
  uint32_t *faults = nullptr;
  uint32_t found = 0;
  auto work = [&]() -> int {
    FOCR_HIP_CHECK(hipMalloc(&lin->gemv_codes, chunks * 16));
    FOCR_HIP_CHECK(hipMalloc(reinterpret_cast<void **>(&lin->gemv_scales), scale_count * sizeof(float)));
    *total += chunks * 16 + scale_count * sizeof(float);
    FOCR_HIP_CHECK(hipMalloc(reinterpret_cast<void **>(&raw), n * k));
    FOCR_HIP_CHECK(hipMalloc(reinterpret_cast<void **>(&faults), sizeof(uint32_t)));
    FOCR_HIP_CHECK(hipMemcpyAsync(raw, codes, n * k, hipMemcpyHostToDevice, ctx->stream));
    FOCR_HIP_CHECK(hipMemcpyAsync(faults, &found, sizeof(uint32_t), hipMemcpyHostToDevice, ctx->stream));
    hipLaunchKernelGGL(pack_kernel, dim3(blocks_for(chunks)), dim3(256), 0, ctx->stream, raw, lin->scales,
                       static_cast<int>(n), static_cast<int>(k), static_cast<int>(lin->group),
                       static_cast<int>(lin->groups), static_cast<int>(steps), chunks,
                       static_cast<uint4 *>(lin->gemv_codes), faults);
    FOCR_HIP_CHECK(hipGetLastError());
    hipLaunchKernelGGL(pack_scales_kernel, dim3(blocks_for(scale_count)), dim3(256), 0, ctx->stream, lin->scales,
                       static_cast<int>(n), static_cast<int>(lin->group), static_cast<int>(lin->groups),
                       static_cast<int>(per), scale_count, lin->gemv_scales);
    FOCR_HIP_CHECK(hipGetLastError());
    if (panels) {
      FOCR_HIP_CHECK(hipMalloc(reinterpret_cast<void **>(&lin->i16_wsum), lin->groups * n * sizeof(int32_t)));
      FOCR_HIP_CHECK(hipMalloc(reinterpret_cast<void **>(&lin->i16_sw), lin->groups * n * sizeof(float)));
      *total += lin->groups * n * (sizeof(int32_t) + sizeof(float));
      hipLaunchKernelGGL(panel_sums_kernel, dim3(static_cast<unsigned>((lin->groups * n + 255) / 256)), dim3(256), 0,
                         ctx->stream, static_cast<const uint8_t *>(lin->gemv_codes), lin->gemv_scales, n, lin->groups,
                         steps, lin->i16_wsum, lin->i16_sw);
      FOCR_HIP_CHECK(hipGetLastError());
    }
    FOCR_HIP_CHECK(hipMemcpyAsync(&found, faults, sizeof(uint32_t), hipMemcpyDeviceToHost, ctx->stream));
    FOCR_HIP_CHECK(hipStreamSynchronize(ctx->stream));
    FOCR_REQUIRE(!(found & 1), FOCR_E_VALUE, "W4 code outside [-8,7]");
    FOCR_REQUIRE(!(found & 2), FOCR_E_VALUE, "nonzero code in zero-scale group");
    return FOCR_OK;
  };
  const int rc = work();
  if (raw) (void)hipFree(raw);
  if (faults) (void)hipFree(faults);
  return rc;
}

int launch_dequantize4(Ctx *ctx, const Linear *lin, float *out) {
  hipLaunchKernelGGL(dequantize4bit_kernel, dim3(blocks_for(lin->n * lin->k)), dim3(256), 0, ctx->stream,
                     static_cast<const uint8_t *>(lin->gemv_codes), lin->gemv_scales, lin->exc_index, lin->exc_vals,
                     static_cast<int>(lin->n_exc), lin->n, lin->k, lin->group, lin->gemv_steps, out);
  FOCR_HIP_CHECK(hipGetLastError());
  return FOCR_OK;
}

int launch_unpack4(Ctx *ctx, const Linear *lin, bool panel, int8_t *out) {
  const dim3 grid(blocks_for(lin->n * lin->k)), block(256);
  const uint8_t *tiles = static_cast<const uint8_t *>(lin->gemv_codes);
  if (panel)
    hipLaunchKernelGGL(unpack_kernel<true>, grid, block, 0, ctx->stream, tiles, lin->n, lin->k, lin->gemv_steps, out);
  else
    hipLaunchKernelGGL(unpack_kernel<false>, grid, block, 0, ctx->stream, tiles, lin->n, lin->k, lin->gemv_steps, out);
  FOCR_HIP_CHECK(hipGetLastError());
  return FOCR_OK;
}

}  // namespace focr
