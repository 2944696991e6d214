// Decode GEMV (1..=8 rows) of 4-bit codes with one FP32 scale per 32, 64 or 128
// input columns, and the kernels around that storage (linear4.hpp): upload,
// dequantization, unpacking for the prefill kernels.
//
//   out[r][n] = epilogue(sum_k x'[r][k] c[n][k] s[n][k / group])
//
// with x' the input row, times a row scale or RMS-normalized if asked.
//
// Mathematics. Each block of 128 W columns of a row of x (W steps of a wave, 1 to 4)
// is written as integers, x = i 2^(e - 22), |i| <= 2^22, 2^e above its largest
// magnitude, and i as three signed bytes, i = d0 + 256 d1 + 65536 d2. Exception columns
// count as zeros in this: their codes are, and their inputs, which may be far larger
// than the others', are added by themselves in FP32. The INT8
// matrix instruction then forms the exact sums of 16 channels' codes times the
// bytes of up to five rows (eight in two instructions) over 64 columns: operands are
// the codes as the tile holds them (no conversion) and the bytes, one column of
// the product per (row, byte). A sum is at most 64 * 128 * 128 = 2^20, so its FP32
// value is exact, and the only roundings are x to 2^(e - 23) and the FP32
// multiply-adds of the groups' sums by their scales. The factor of a row (its scale,
// or its RMS norm's, whose sum of squares is taken as the row goes by) multiplies
// the finished sums. A row that holds an infinity or NaN is marked, and
// its outputs, infinities and NaNs all, are found from those inputs after the others
// (24,576 x 8,192 for eight rows: 31.8 us, 32.7 with a row of NaNs, 43.7 with an infinity).
#include <type_traits>

#include "linear4.hpp"

namespace focr {
namespace {

using namespace linear4;

typedef int v4i __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v4f_apart __attribute__((ext_vector_type(4), aligned(4)));

constexpr int kWaves = 8;
constexpr size_t kLdsBytes = 160 * 1024;

struct Args {
  const uint4 *tiles;
  const float *scales;
  const int32_t *exc_cols;
  const float *exc_vals;
  const int16_t *exc_index;  // [k up to whole fours]: below 0 where a column is no exception; null: none
  int n_exc;
  const float *x, *row_scale;
  float *out;
  int m, n, k, group, steps, tiles_total, rms, epilogue;
  // The rows as they are staged: x, but for rows of fewer than four columns, which are
  // computed like those with an infinity (plain).
  const float *staged;
  int staged_k;
  uint32_t plain;
  // What rows4_kernel writes (PRE): the blocks and their weights as they stand in the
  // GEMV's LDS, sums of squares [8][blocks] and non-finite marks [8][blocks].
  char *digits;
  float *weights, *squares;
  uint32_t *marks;
  int blocks;
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

// The largest of a wave, in every lane.
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  v = row_max16(v);
  const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = a[0] > a[1] ? a[0] : a[1];
  const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return b[0] > b[1] ? b[0] : b[1];
}

// The sum over a wave, in every lane.
__device__ __forceinline__ float wave_sum(float v) {
  v = v + row_up<8>(v);
  v = v + row_up<4>(v);
  v = v + row_up<2>(v);
  v = v + row_up<1>(v);
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// A load at a uniform address and a lane's offset: one register of it, not two.
template <typename T>
__device__ __forceinline__ T load_at(const void *base, uint32_t offset) {
  return *reinterpret_cast<const T *>(static_cast<const char *>(base) + offset);
}

// Four columns of row r (the same for the wave) in one load, which needs no more than
// FP32's alignment: the row's last four past its end, `trim`med when they are used.
__device__ __forceinline__ v4f load_x(const Args &a, int r, int col) {
  return load_at<v4f_apart>(a.staged + static_cast<size_t>(r) * a.staged_k, 4u * (col < a.staged_k - 4 ? col : a.staged_k - 4));
}
// Their values: zeros past the row's end.
__device__ __forceinline__ v4f trim(const Args &a, v4f v, int col) {
  const int k = a.staged_k, over = col - (k - 4);  // positions that the load went back
  if (k % 4 != 0) {
    v = over == 1 ? v4f{v[1], v[2], v[3], 0.0f} : over == 2 ? v4f{v[2], v[3], 0.0f, 0.0f} : over == 3 ? v4f{v[3], 0.0f, 0.0f, 0.0f} : v;
  }
  return over < 4 ? v : v4f{0.0f, 0.0f, 0.0f, 0.0f};
}

// 1 / sqrt(mean of squares + eps) from the sum of squares.
__device__ __forceinline__ float rms_factor(float sum, int k) {
  return __fdiv_rn(1.0f, __builtin_sqrtf(__fdiv_rn(sum, static_cast<float>(k)) + 1.1920929e-7f));
}
__device__ __forceinline__ float square_sum(v4f v, float sum) {
#pragma unroll
  for (int i = 0; i < 4; i++) sum = fmaf_(v[i], v[i], sum);
  return sum;
}

// The product's columns: with one 16-column block column 5 d + r holds byte d of
// row r (5 rows), with two column 8 d + r (8 rows).
template <int NB>
struct Columns {
  static constexpr int kWide = 16 * NB, kRows = NB == 1 ? 5 : 8;
  // A 64-column group: [4 lane chunks][columns][16 bytes].
  static constexpr int kGroup = 64 * kWide;
  __device__ static __forceinline__ int at(int kg, int col) { return (kg * kWide + col) * 16; }
};

// A block of 128 W columns of a row in a wave's registers, 256 columns at a time.
template <int W>
struct Block {
  static constexpr int kParts = (W + 1) / 2;
  v4f v[kParts];
  __device__ static __forceinline__ bool holds(int p) { return 2 * p + (threadIdx.x & 63) / 32 < W; }
  // Columns past the block's count as past the row.
  __device__ static __forceinline__ int column(const Args &a, int col0, int p) {
    return holds(p) ? col0 + 256 * p + 4 * (threadIdx.x & 63) : a.staged_k;
  }
  __device__ __forceinline__ void load(const Args &a, int r, int col0) {
#pragma unroll
    for (int p = 0; p < kParts; p++) v[p] = load_x(a, r, column(a, col0, p));
  }
  // Which of the lane's columns are exceptions: bit 4 p + i, the same for all rows.
  __device__ static __forceinline__ uint32_t exceptions(const Args &a, int col0) {
    uint32_t marks = 0;
    if (a.exc_index) {
      const int last = (a.staged_k - 1) / 4 * 4;
#pragma unroll
      for (int p = 0; p < kParts; p++) {
        const int col = column(a, col0, p);
        const uint2 index = load_at<uint2>(a.exc_index, 2u * (col < last ? col : last));
        marks |= ((~index.x >> 15 & 1) | (~index.x >> 30 & 2) | (~index.y >> 13 & 4) | (~index.y >> 28 & 8)) << (4 * p);
      }
    }
    return marks;
  }
  __device__ __forceinline__ void trim_to(const Args &a, int col0) {
#pragma unroll
    for (int p = 0; p < kParts; p++) v[p] = trim(a, v[p], column(a, col0, p));
  }
};

// A wave writes block x of row r: bytes to `digits` [2 W groups], their weights to
// `weights` [columns]; exceptions become zeros. True (in every lane) if a value is not
// finite.
template <int NB, int W>
__device__ __forceinline__ bool stage_block(Block<W> &x, uint32_t exceptions, int r, char *digits, float *weights) {
  using C = Columns<NB>;
  constexpr int P = Block<W>::kParts;
  const int lane = threadIdx.x & 63, l16 = lane & 15;
  v4f(&v)[P] = x.v;
  bool outlier = false;  // an exception that is not finite
  if (__any(exceptions != 0)) {
#pragma unroll
    for (int p = 0; p < P; p++) {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const bool taken = exceptions >> (4 * p + i) & 1;
        outlier |= taken && (__float_as_uint(v[p][i]) & 0x7fffffffu) >= 0x7f800000u;
        v[p][i] = taken ? 0.0f : v[p][i];
      }
    }
    outlier = __any(outlier);
  }
  uint32_t big = 0;
#pragma unroll
  for (int p = 0; p < P; p++) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint32_t bits = __float_as_uint(v[p][i]) & 0x7fffffffu;
      big = bits > big ? bits : big;
    }
  }
  big = wave_max(big);
  const bool bad = big >= 0x7f800000u;
  int e = bad || big == 0 ? 0 : __builtin_amdgcn_frexp_expf(__uint_as_float(big));
  e = e < -96 ? -96 : e;
  // 1.5 2^23 + i holds the integer i in its low bits; adding 128 to each byte of
  // i and inverting their top bits leaves signed bytes whose weighted sum is i.
  auto bytes = [&](float f) {
    const float t = __builtin_ldexpf(f, 22 - e) + 12582912.0f;
    return (__float_as_uint(t) + (0x00808080u - 0x4b400000u)) ^ 0x00808080u;
  };
#pragma unroll
  for (int p = 0; p < P; p++) {
    const uint32_t w0 = bytes(v[p][0]), w1 = bytes(v[p][1]), w2 = bytes(v[p][2]), w3 = bytes(v[p][3]);
    const uint32_t a01 = __builtin_amdgcn_perm(w1, w0, 0x05010400u), a23 = __builtin_amdgcn_perm(w3, w2, 0x05010400u);
    const uint32_t b01 = __builtin_amdgcn_perm(w1, w0, 0x0c0c0602u), b23 = __builtin_amdgcn_perm(w3, w2, 0x0c0c0602u);
    const uint32_t d[3] = {__builtin_amdgcn_perm(a23, a01, 0x05040100u), __builtin_amdgcn_perm(a23, a01, 0x07060302u),
                           __builtin_amdgcn_perm(b23, b01, 0x05040100u)};
    if (x.holds(p)) {
      char *to = digits + (4 * p + lane / 16) * C::kGroup + C::at(l16 / 4, r) + 4 * (l16 % 4);
#pragma unroll
      for (int i = 0; i < 3; i++) *reinterpret_cast<uint32_t *>(to + i * C::kRows * 16) = d[i];
    }
  }
  if (lane < 3) weights[lane * C::kRows + r] = __builtin_ldexpf(1.0f, e - 26 + 8 * lane);
  return bad || outlier;
}

// The rows as bytes in memory, for large calls: a wave for each block of a row.
// Bound by its launch: eight rows of 8,192 take 3.2 us and move 0.7 MB.
template <int NB, int W>
__global__ __launch_bounds__(256) void rows4_kernel(Args a) {
  using C = Columns<NB>;
  const int r = blockIdx.y, block = 4 * blockIdx.x + threadIdx.x / 64;
  if (block >= a.blocks) return;
  Block<W> x;
  x.load(a, r, block * W * kStep);
  const uint32_t exceptions = Block<W>::exceptions(a, block * W * kStep);
  x.trim_to(a, block * W * kStep);
  float sum = 0.0f;
#pragma unroll
  for (int p = 0; p < Block<W>::kParts; p++) sum = square_sum(x.v[p], sum);
  sum = wave_sum(sum);
  const bool bad = stage_block<NB, W>(x, exceptions, r, a.digits + static_cast<size_t>(block) * 2 * W * C::kGroup,
                                      a.weights + block * C::kWide);
  if (threadIdx.x % 64 == 0) {
    a.marks[r * a.blocks + block] = bad;
    a.squares[r * a.blocks + block] = sum;
  }
}

// The workgroup's LDS accesses so far, and no load from memory, are waited for.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Waves of a SIMD that the registers leave room for: two workgroups of a compute
// unit, or one where LDS holds no more (or the scales of 32 columns take the registers).
template <int NB, int SK, int W, int G, bool PRE>
constexpr int resident() {
  return (G == 32 && W > 2) || (PRE ? 2 : 1) * SK * 2 * W * Columns<NB>::kGroup > 80 * 1024 ? 2 : 4;
}

// NB: 16-column blocks of the product (Columns). SK: waves that share a tile's
// columns, each W steps of a turn. G: columns per scale. PRE: the rows come as bytes
// from rows4_kernel and pass through LDS turn by turn; otherwise the workgroup
// writes all of them to LDS itself. NW: waves of a workgroup.
// Bound: the codes, read once. A wave's load is 1 KB, a tile's step, and W of them
// with their scales are on their way while W others are used; a load under a branch,
// or a spilled register, would make the wave wait for all of them. 24,576 x 8,192 in
// groups of 64 take 26.1 us for eight rows (114 MB, 4.4 TB/s), 65,536 x 768 in groups
// of 128 7.7 us for one (27 MB, 3.5 TB/s: a third of it is the launch and the rows);
// 2,048 x 768 take 4.7 us, all launch, rows and one trip to memory.
template <int NB, int SK, int W, int G, bool PRE, int NW>
__global__ __launch_bounds__(64 * NW, (resident<NB, SK, W, G, PRE>())) void gemv4_kernel(Args a) {
  using C = Columns<NB>;
  constexpr int NS = kStep / G;             // scales of a channel per step
  constexpr int SLOTS = NW / SK;        // tiles a workgroup has at once
  constexpr int BLOCK = 2 * W * C::kGroup;  // bytes of a block
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int steps = a.steps, M = a.m, k = a.k;
  const int turns = (steps + W * SK - 1) / (W * SK);
  const int held = PRE ? 2 * SK : turns * SK;                          // blocks in LDS
  float *const weights = reinterpret_cast<float *>(lds + held * BLOCK);  // [held][columns]
  float *const red = weights + held * C::kWide;                         // [NW][8][16]
  float *const squares = red + NW * 8 * 16;                         // [8][SK]
  uint32_t *const bad = reinterpret_cast<uint32_t *>(squares + 8 * SK);  // [8]
  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, kg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int slot = wave / SK, part = wave % SK;

  // The wave's work: of tiles first, first + stride, ... block part of every
  // turn: W steps, whose bytes are zeros past the last one.
  const int stride = gridDim.x * SLOTS;
  const int rounds = (a.tiles_total + stride - 1) / stride;
  v4u codes[W];
  v4f scales[W][NS];
  auto load = [&](int i, int round, int turn) {
    int tile = slot + SLOTS * blockIdx.x + round * stride;
    tile = tile < a.tiles_total ? tile : a.tiles_total - 1;
    int step = (turn * SK + part) * W + i;
    step = step < steps ? step : steps - 1;
    const size_t at = static_cast<size_t>(tile) * steps + step;
    codes[i] = load_at<v4u>(a.tiles + at * 64, 16u * lane);
#pragma unroll
    for (int q = 0; q < NS; q++) scales[i][q] = load_at<v4f>(a.scales + (at * NS + q) * kTile, 16u * kg);
  };

  // PRE: a turn's bytes from memory to registers and on to LDS, and its weights to
  // registers.
  constexpr int PIECES = SK * BLOCK / 16;  // 16 bytes each
  constexpr int PER = PRE ? (PIECES + 64 * NW - 1) / (64 * NW) : 1;
  static_assert(!PRE || PIECES >= 64 * NW, "a piece for each thread");
  v4u moved[PER];
  float weight[NB];
  // A thread with no piece left moves its last one again: no branch, no wait in one.
  auto piece_of = [&](int p) {
    const int piece = tid + 64 * NW * p;
    return piece < PIECES ? piece : piece - 64 * NW;
  };
  auto fetch = [&](int turn) {
#pragma unroll
    for (int p = 0; p < PER; p++) moved[p] = load_at<v4u>(a.digits + static_cast<size_t>(turn) * PIECES * 16, 16u * piece_of(p));
  };
  auto fetch_weight = [&](int turn) {
#pragma unroll
    for (int b = 0; b < NB; b++) weight[b] = a.weights[(turn * SK + part) * C::kWide + 16 * b + l16];
  };
  auto place = [&](int buffer) {
#pragma unroll
    for (int p = 0; p < PER; p++) reinterpret_cast<v4u *>(lds)[buffer * PIECES + piece_of(p)] = moved[p];
  };
  if constexpr (PRE) {
    fetch(0);
    fetch_weight(0);
#pragma unroll
    for (int i = 0; i < W; i++) load(i, 0, 0);
    // A wave sums a row's squares and marks over its blocks.
    for (int r = wave; r < M; r += NW) {
      float sum = 0.0f;
      uint32_t any = 0;
      for (int block = lane; block < a.blocks; block += 64) {
        sum = sum + a.squares[r * a.blocks + block];
        any |= a.marks[r * a.blocks + block];
      }
      sum = wave_sum(sum);
      const bool found = __any(any != 0);
      if (lane < SK) squares[r * SK + lane] = lane == 0 ? sum : 0.0f;
      if (lane == 0) bad[r] = found;
    }
    place(0);
    lds_barrier();
  } else {
    // The rows' loads go before the codes': loads arrive in order, and so the rows
    // are written while the codes are on their way. This wave writes block
    // turn * SK + part of rows slot, slot + SLOTS, ...
    constexpr int ROWS = (C::kRows + SLOTS - 1) / SLOTS;
    Block<W> x[ROWS];
    float sum[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; i++) sum[i] = 0.0f;
    uint32_t exceptions = 0;
    // Past the call's rows, the last one again (not written).
    auto load_rows = [&](int turn) {
#pragma unroll
      for (int i = 0; i < ROWS; i++) {
        const int r = slot + SLOTS * i;
        x[i].load(a, r < M ? r : M - 1, (turn * SK + part) * W * kStep);
      }
      exceptions = Block<W>::exceptions(a, (turn * SK + part) * W * kStep);
    };
    load_rows(0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < W; i++) load(i, 0, 0);
    __builtin_amdgcn_sched_barrier(0);
    if (tid < 8) bad[tid] = a.plain;
    lds_barrier();
    for (int turn = 0; turn < turns; turn++) {
      if (turn > 0) load_rows(turn);
      const int block = turn * SK + part;
#pragma unroll
      for (int i = 0; i < ROWS; i++) {
        const int r = slot + SLOTS * i;
        if (r >= M) continue;
        x[i].trim_to(a, block * W * kStep);
        if (a.rms)
#pragma unroll
          for (int p = 0; p < Block<W>::kParts; p++) sum[i] = square_sum(x[i].v[p], sum[i]);
        if (stage_block<NB, W>(x[i], exceptions, r, lds + block * BLOCK, weights + block * C::kWide)) bad[r] = 1;
      }
    }
    // The rows' sums of squares by waves, for `finish`.
    if (a.rms)
#pragma unroll
      for (int i = 0; i < ROWS; i++) {
        const float total = wave_sum(sum[i]);
        if (lane == 0 && slot + SLOTS * i < M) squares[(slot + SLOTS * i) * SK + part] = total;
      }
    lds_barrier();
  }

  float acc[NB][4];
#pragma unroll
  for (int b = 0; b < NB; b++)
#pragma unroll
    for (int i = 0; i < 4; i++) acc[b][i] = 0.0f;
  // Step i of the block at `digits`, added to the block's sums.
  auto consume = [&](const v4u &word, const v4f(&s)[NS], const char *digits, float(&sum)[NB][4]) {
#pragma unroll
    for (int half = 0; half < 2; half++) {
      v4i A;
#pragma unroll
      for (int w = 0; w < 2; w++) {
        A[2 * w] = static_cast<int>((word[2 * half + w] << 4) & 0xf0f0f0f0u);
        A[2 * w + 1] = static_cast<int>(word[2 * half + w] & 0xf0f0f0f0u);
      }
#pragma unroll
      for (int b = 0; b < NB; b++) {
        const v4i B = *reinterpret_cast<const v4i *>(digits + half * C::kGroup + C::at(kg, 16 * b + l16));
        const v4i zero = {0, 0, 0, 0};
        auto add = [&](const v4i &c, const v4f &q) {
#pragma unroll
          for (int i = 0; i < 4; i++) sum[b][i] = fmaf_(static_cast<float>(c[i]), q[i], sum[b][i]);
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

  // What an ADD call adds to: loaded ahead of a tile's last turn.
  const bool quads = a.n % 4 == 0 && (reinterpret_cast<uintptr_t>(a.out) & 15) == 0;
  v4f residual = {0.0f, 0.0f, 0.0f, 0.0f};
  auto load_residual = [&](int round) {
    const int ch = (slot + SLOTS * blockIdx.x + round * stride) * kTile + 4 * kg;
    if (l16 >= M || part > 0 || ch >= a.n) return;
    const float *out = a.out + static_cast<size_t>(l16) * a.n + ch;
    if (quads) {
      residual = *reinterpret_cast<const v4f *>(out);
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++) residual[i] = out[ch + i < a.n ? i : 0];
    }
  };

  // A row's scale, or its norm's.
  const bool scaled = a.rms || a.row_scale;
  auto row_factor = [&](int r) {
    if (!a.rms) return a.row_scale ? a.row_scale[r] : 1.0f;
    float total = squares[r * SK];
#pragma unroll
    for (int p = 1; p < SK; p++) total += squares[r * SK + p];
    return rms_factor(total, k);
  };

  // The rows of a finished tile that are not marked: lane l16 = row, channels 4 kg .. + 3.
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
      lds_barrier();
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
      lds_barrier();
      if (part > 0) return;
    }
    const int r = l16, ch = tile * kTile + 4 * kg;
    if (r >= M || tile >= a.tiles_total || ch >= a.n || bad[r]) return;
    const float *row = a.x + static_cast<size_t>(r) * k;
    const float factor = row_factor(r);
    if (scaled)
#pragma unroll
      for (int i = 0; i < 4; i++) total[i] = total[i] * factor;
    auto x_at = [&](int col) { return scaled ? row[col] * factor : row[col]; };
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
    if (a.epilogue == FOCR_EPI_ADD)
#pragma unroll
      for (int i = 0; i < 4; i++) total[i] = residual[i] + total[i];
    float *out = a.out + static_cast<size_t>(r) * a.n + ch;
    if (quads) {
      *reinterpret_cast<v4f *>(out) = v4f{total[0], total[1], total[2], total[3]};
      return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (ch + i < a.n) out[i] = total[i];
  };

  // Turn after turn: every load is one that the next turn consumes, and none is
  // under a branch, so a step waits for its own codes only. A turn with nothing
  // after it loads nothing.
  int round = 0, turn = 0, buffer = 0;
  auto take = [&](auto more) {
    constexpr bool kMore = decltype(more)::value;
    const bool ends = turn + 1 == turns;
    const int next_round = ends ? round + 1 : round, next_turn = ends ? 0 : turn + 1;
    if (ends && a.epilogue == FOCR_EPI_ADD) load_residual(round);
    if constexpr (PRE && kMore) fetch(next_turn);
    const int block = PRE ? buffer * SK + part : turn * SK + part;
    float block_sum[NB][4], f[NB];
#pragma unroll
    for (int b = 0; b < NB; b++) {
      f[b] = PRE ? weight[b] : weights[block * C::kWide + 16 * b + l16];
#pragma unroll
      for (int i = 0; i < 4; i++) block_sum[b][i] = 0.0f;
    }
    if constexpr (PRE && kMore) fetch_weight(next_turn);
#pragma unroll
    for (int i = 0; i < W; i++) {
      consume(codes[i], scales[i], lds + block * BLOCK + 2 * i * C::kGroup, block_sum);
      if constexpr (kMore) load(i, next_round, next_turn);
    }
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
      for (int i = 0; i < 4; i++) acc[b][i] = fmaf_(block_sum[b][i], f[b], acc[b][i]);
    if constexpr (PRE && kMore) {
      buffer ^= 1;
      place(buffer);
      lds_barrier();
    }
    if (ends) finish(round);
    round = next_round;
    turn = next_turn;
  };
  for (int t = 1; t < rounds * turns; t++) take(std::true_type());
  take(std::false_type());

  // Marked rows, with the loads above out of the way: lane l16 = channel. A NaN, or an
  // infinity times a norm's factor (zero then), makes all of a row NaN; otherwise the
  // products with its infinities are its sums, whatever the finite ones are. The lanes
  // look for them together, four columns each. (Plain rows: all columns.)
  for (unsigned long long marked = part > 0 ? 0 : __ballot(lane < M && bad[lane & 7]); marked; marked &= marked - 1) {
    const int r = __ffsll(marked) - 1;
    const float *row = a.x + static_cast<size_t>(r) * k;
    float factor;
    if (a.rms && a.plain) {
      float total = 0.0f;
      for (int col = 0; col < k; col++) total = fmaf_(row[col], row[col], total);
      factor = rms_factor(total, k);
    } else {
      factor = row_factor(r);
    }
    auto x_at = [&](int col) { return scaled ? row[col] * factor : row[col]; };
    for (int now = 0; now < rounds; now++) {
      const int tile = slot + SLOTS * blockIdx.x + now * stride, ch = tile * kTile + l16;
      if (tile >= a.tiles_total) break;
      float total = 0.0f;
      bool nan = a.rms && !a.plain;
      auto add = [&](int col) {
        if (col < k && (a.plain || __builtin_fabsf(row[col]) == __builtin_inff()))
          total = fmaf_(x_at(col),
                        static_cast<float>(code_at(reinterpret_cast<const uint8_t *>(a.tiles), steps, ch, col)) *
                            scale_at(a.scales, steps, G, ch, col),
                        total);
      };
      for (int col = 0; a.plain && col < k; col++) add(col);
      for (int col0 = 0; !a.plain && !nan && col0 < k; col0 += 256) {
        const v4f v = trim(a, load_x(a, r, col0 + 4 * lane), col0 + 4 * lane);
        nan = __any(v[0] != v[0] || v[1] != v[1] || v[2] != v[2] || v[3] != v[3]);
        const float most = __builtin_fmaxf(__builtin_fmaxf(__builtin_fabsf(v[0]), __builtin_fabsf(v[1])),
                                           __builtin_fmaxf(__builtin_fabsf(v[2]), __builtin_fabsf(v[3])));
        for (unsigned long long found = __ballot(most == __builtin_inff()); found && !nan; found &= found - 1) {
          const int first = col0 + 4 * (__ffsll(found) - 1);
          for (int col = first; col < first + 4; col++) add(col);
          nan = !__any(total == total);
        }
      }
      if (nan) total = __builtin_nanf("");
      for (int e = 0; e < a.n_exc; e++)
        if (ch < a.n) total = fmaf_(x_at(a.exc_cols[e]), a.exc_vals[static_cast<size_t>(ch) * a.n_exc + e], total);
      const float up = __shfl_xor(total, 1);
      if (kg > 0 || ch >= a.n) continue;
      float *out = a.out + static_cast<size_t>(r) * a.n + ch;
      if (a.epilogue == FOCR_EPI_GLU) {
        if (l16 % 2 == 0) a.out[static_cast<size_t>(r) * (a.n / 2) + ch / 2] = squared_relu_glu(total, up);
      } else {
        *out = a.epilogue == FOCR_EPI_ADD ? *out + total : total;
      }
    }
  }
}

// Turns of a row, and the fewest steps of a turn that take all of it in them.
constexpr int turns_of(int steps, int sk) { return (steps + 4 * sk - 1) / (4 * sk); }
constexpr int width_of(int steps, int sk) {
  const int turns = turns_of(steps, sk);
  return (steps + sk * turns - 1) / (sk * turns);
}
// LDS of a workgroup.
size_t lds_of(int nb, int sk, int w, size_t held) {
  return held * (2 * w * 64 * 16 * nb + 16 * nb * 4) + kWaves * 8 * 16 * 4 + 8 * sk * 4 + 8 * 4;
}

template <int NB, int SK, int W, int G, bool PRE, int NW = kWaves>
int launch_one(Ctx *ctx, const Args &a) {
  if constexpr (PRE) {
    hipLaunchKernelGGL((rows4_kernel<NB, W>), dim3((a.blocks + 3) / 4, a.m), dim3(256), 0, ctx->stream, a);
    FOCR_HIP_CHECK(hipGetLastError());
  }
  const size_t turns = (a.steps + W * SK - 1) / (W * SK), lds = lds_of(NB, SK, W, PRE ? 2 * SK : turns * SK);
  FOCR_REQUIRE(lds <= kLdsBytes, FOCR_E_SHAPE, "GEMV: the rows of x exceed LDS");
  // Above 64 KB the kernel has to be allowed it, on each device.
  if (lds > 64 * 1024)
    FOCR_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void *>(gemv4_kernel<NB, SK, W, G, PRE, NW>),
                                       hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kLdsBytes)));
  constexpr int slots = NW / SK;
  const int want = (a.tiles_total + slots - 1) / slots;
  const int most = lds > kLdsBytes / 2 ? 256 : 512;  // workgroups that 256 compute units hold at once
  const int blocks = want < most ? want : most;
  hipLaunchKernelGGL((gemv4_kernel<NB, SK, W, G, PRE, NW>), dim3(blocks), dim3(64 * NW), lds, ctx->stream, a);
  FOCR_HIP_CHECK(hipGetLastError());
  return FOCR_OK;
}

template <int NB, int SK, int G>
int launch_steps(Ctx *ctx, const Args &a) {
  switch (width_of(a.steps, SK)) {
    case 1: return launch_one<NB, SK, 1, G, false>(ctx, a);
    case 2: return launch_one<NB, SK, 2, G, false>(ctx, a);
    case 3: return launch_one<NB, SK, 3, G, false>(ctx, a);
    default: return launch_one<NB, SK, 4, G, false>(ctx, a);
  }
}
// Rows as bytes: more than one turn, so that W is 3 or 4 (one wave a tile: many
// turns, and 4).
template <int NB, int SK, int G>
int launch_pre(Ctx *ctx, Args a) {
  using C = Columns<NB>;
  const int turns = turns_of(a.steps, SK) < 2 ? 2 : turns_of(a.steps, SK);
  const int w = SK > 1 && (a.steps + SK * turns - 1) / (SK * turns) <= 3 ? 3 : 4;
  const size_t blocks = static_cast<size_t>((a.steps + w * SK - 1) / (w * SK)) * SK;
  const size_t digits = blocks * 2 * w * C::kGroup;
  const int rc = ensure_scratch(ctx, digits + blocks * (C::kWide * 4 + 8 * 4 + 8 * 4));
  if (rc != FOCR_OK) return rc;
  a.blocks = static_cast<int>(blocks);
  a.digits = static_cast<char *>(ctx->scratch);
  a.weights = reinterpret_cast<float *>(a.digits + digits);
  a.squares = a.weights + blocks * C::kWide;
  a.marks = reinterpret_cast<uint32_t *>(a.squares + 8 * blocks);
  if constexpr (SK > 1) {
    if (w == 3) return launch_one<NB, SK, 3, G, true>(ctx, a);
  } else if constexpr (NB == 1) {
    // The tiles of the busiest compute unit, with workgroups of eight tiles or of six
    // (us with eight / six: 24,576 x 8,192 for five rows 30.3 / 27.5, 40,000 x 5,000
    // for four 32.9 / 29.9; for more than five rows the products leave no gain, 32.9
    // / 33.5).
    auto busiest = [&](int nw) {
      const int groups = (a.tiles_total + nw - 1) / nw;
      return groups > 512 ? a.tiles_total : (groups + 255) / 256 * nw;
    };
    if (busiest(6) < busiest(8)) return launch_one<NB, SK, 4, G, true, 6>(ctx, a);
  }
  return launch_one<NB, SK, 4, G, true>(ctx, a);
}

// Few tiles are shared by many waves, so that every SIMD has work: 4,096 x 8,192 for
// one row takes 8.4 us with eight waves a tile and 14.4 with two, and 27,807 x 2,132
// for two rows 12.8 with two and 15.5 with four. Bytes from memory reach LDS once for
// a turn of all the workgroup's tiles, so that half as many waves a tile are right
// there: 20,000 x 5,000 for four rows takes 15.5 us with one and 16.7 with two.
constexpr int waves_of(int tiles) { return tiles >= 1024 ? 2 : tiles >= 512 ? 4 : 8; }

// Above this many columns in all rows a kernel of its own writes their bytes once:
// at 32,768 columns 11,008 channels take 11.9 us with it and 14.2 with the rows
// written by every workgroup; a launch more costs what 16,384 columns gain (8,192
// channels: 7.2 us without it, 4,096: 6.9 without it and 9.5 with it).
constexpr long kPreColumns = 16384;

template <int NB, int G>
int launch_parts(Ctx *ctx, const Args &a) {
  const int sk = waves_of(a.tiles_total);
  const size_t lds = lds_of(NB, sk, width_of(a.steps, sk), static_cast<size_t>(turns_of(a.steps, sk)) * sk);
  const bool pre = static_cast<long>(a.m) * a.k > kPreColumns || lds > kLdsBytes;
  if (sk == 2) return pre ? launch_pre<NB, 1, G>(ctx, a) : launch_steps<NB, 2, G>(ctx, a);
  if (sk == 4) return pre ? launch_pre<NB, 2, G>(ctx, a) : launch_steps<NB, 4, G>(ctx, a);
  return pre ? launch_pre<NB, 4, G>(ctx, a) : launch_steps<NB, 8, G>(ctx, a);
}

template <int NB>
int launch_group(Ctx *ctx, const Args &a) {
  switch (a.group) {
    case 32: return launch_parts<NB, 32>(ctx, a);
    case 64: return launch_parts<NB, 64>(ctx, a);
    default: return launch_parts<NB, 128>(ctx, a);
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
  const size_t steps = steps_of(lin->k);
  Args a = {};
  a.tiles = static_cast<const uint4 *>(lin->gemv_codes);
  a.scales = lin->gemv_scales;
  a.exc_cols = lin->exc_cols;
  a.exc_vals = lin->exc_vals;
  a.exc_index = lin->n_exc ? lin->exc_index : nullptr;
  a.n_exc = static_cast<int>(lin->n_exc);
  a.x = x;
  a.row_scale = row_scale;
  a.out = out;
  a.m = static_cast<int>(rows);
  a.n = static_cast<int>(lin->n);
  a.k = static_cast<int>(lin->k);
  a.group = static_cast<int>(lin->group);
  a.steps = static_cast<int>(steps);
  a.tiles_total = static_cast<int>(lin->gemv_tiles);
  a.rms = rms_norm ? 1 : 0;
  a.epilogue = epilogue;
  a.staged = lin->k < 4 ? lin->gemv_scales : x;  // 16 floats at least
  a.staged_k = lin->k < 4 ? 4 : a.k;
  a.plain = lin->k < 4;
  if (a.plain && a.m > 1) {
    // One row at a time: the scales of one tile are the rows.
    for (size_t r = 0; r < rows; r++) {
      Args one = a;
      one.m = 1;
      one.x = x + r * lin->k;
      one.row_scale = row_scale ? row_scale + r : nullptr;
      one.out = out + r * (epilogue == FOCR_EPI_GLU ? lin->n / 2 : lin->n);
      const int rc = launch_group<1>(ctx, one);
      if (rc != FOCR_OK) return rc;
    }
    return FOCR_OK;
  }
  return rows <= 5 ? launch_group<1>(ctx, a) : launch_group<2>(ctx, a);
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
