// A cache of pages that sequences share, in 8 bits: appending a step's keys and
// values (ready, or split, normalized and rotated from the QKV rows on the way),
// attention of 1..=8 rows of every sequence of a batch, and reading rows back.
//
// A block is 16 positions of one head: 1 KB of codes and one FP32 scale,
//
//   scale = fl(m / 127), m the largest magnitude of the block's stored positions
//   code = rint(fl(x fl(1 / scale))), and the block holds fl(code scale)
//
// (zeros where m / 127 is below 2^-126; NaN where a value is not finite). Pages hold
// `page` positions, a power of two from 16 on: for each head its blocks in order.
// Key codes stand as [position % 4][position / 4][64], value codes as
// [dim][16 positions]: what the attention's matrix instructions take 16 bytes at a
// time, in runs of 256 bytes for a load of a wave.
//
// A block that is not full is written again by the next append, with the scale that
// its positions then need. So that this rounds every value once, the last two
// blocks of a sequence are also kept in FP32 beside the pages (two, so that a step
// that takes back up to 16 positions finds them too): what the cache holds depends
// on the rows appended, and not on how many at a time. Where a block is not
// there (a sequence that goes on from pages it was given, or goes back further), or
// another sequence wrote the page's block since, its earlier positions are taken from
// its codes.
#include <algorithm>
#include <new>
#include <type_traits>

#include "decode_common.hpp"
#include "rms_tree.hpp"
#include "rotary.hpp"

namespace focr {
namespace {

constexpr int kBlock = 16, kBlockBytes = kBlock * 64;

typedef int v4i __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));

struct Pages {
  int device = 0, shift = 0;  // log2 of the blocks of a page
  size_t n_pages = 0, page = 0, n_seqs = 0, seq_pages = 0, n_heads = 0, key_heads = 0, kv_heads = 0;
  int8_t *k_codes = nullptr;   // [page][key head][block][1 KB]
  int8_t *v_codes = nullptr;   // [page][KV head][block][1 KB]
  float *k_scales = nullptr, *v_scales = nullptr;  // [page][head][block]
  int32_t *k_writers = nullptr, *v_writers = nullptr;  // [page][head][block]: the sequence that wrote it, or -1
  int32_t *table = nullptr;    // [sequence][seq_pages], -1: no page
  float *open = nullptr;       // [sequence][key heads, then KV heads][block % 2][16][64]
  int32_t *tags = nullptr;     // [sequence][heads][2]: the block that `open` holds, or -1
  int32_t *refused = nullptr;  // [sequence]
  size_t device_bytes = 0;
};

// What the kernels read of a cache, and a call's rows.
struct Cache {
  int8_t *k_codes, *v_codes;
  float *k_scales, *v_scales;
  int32_t *k_writers, *v_writers;
  const int32_t *table;
  float *open;
  int32_t *tags, *refused;
  int shift, seq_pages, n_heads, key_heads, kv_heads;
  const int32_t *row_start, *lens;  // row_start null: row r is sequence r's
  int rows, n_seqs;

  // Positions `len` .. `len + n - 1` of a sequence are rows `first` .. of the call;
  // false if it is refused (n and len are 0 then, as for one that takes no part).
  __device__ __forceinline__ bool span(int seq, int &len, int &first, int &n) const {
    first = row_start ? row_start[seq] : seq;
    const int end = row_start ? row_start[seq + 1] : seq + 1;
    len = lens[seq];
    n = end - first;
    if (len < 0) {
      n = len = 0;
      return true;
    }
    const long capacity = static_cast<long>(seq_pages) << (shift + 4);
    if (first < 0 || end < first || end > rows || static_cast<long>(len) + n > capacity) {
      n = len = 0;
      return false;
    }
    return true;
  }
  // The block's number in the pages of one head, or -1 if it has no page.
  __device__ __forceinline__ long block_at(int seq, int block, int heads, int head) const {
    const int page = table[static_cast<size_t>(seq) * seq_pages + (block >> shift)];
    return page < 0 ? -1 : (((static_cast<long>(page) * heads + head) << shift) + (block & ((1 << shift) - 1)));
  }
};

// One unit of a call's work that is dealt over the sequences: `of` gives the units of
// n rows from position len on. A wave finds unit u; false past the last one. Rows
// have to begin where the sequences before end, or later, so that all units together
// are bounded by the call's rows.
struct Unit {
  int seq, len, first, n, index;
};
template <typename Of>
__device__ __forceinline__ bool find_unit(const Cache &c, int u, const Of &of, Unit &unit) {
  const int lane = threadIdx.x & 63;
  if (!c.row_start) {
    if (u >= c.n_seqs) return false;
    unit.seq = u;
    unit.index = 0;
    if (!c.span(u, unit.len, unit.first, unit.n)) c.refused[u] = 1;
    return unit.n > 0;
  }
  int before = 0, most = 0;
  for (int base = 0; base < c.n_seqs; base += 64) {
    const int seq = base + lane;
    int len = 0, first = 0, n = 0, units = 0, reach = 0;
    bool fine = true;
    if (seq < c.n_seqs) {
      fine = c.span(seq, len, first, n);
      reach = n > 0 ? first + n : 0;
    }
    // The furthest end of the sequences before this one.
    int top = reach;
    for (int d = 1; d < 64; d *= 2) {
      const int o = __shfl_up(top, d);
      if (lane >= d) top = o > top ? o : top;
    }
    int prior = __shfl_up(top, 1);
    prior = lane == 0 ? most : (prior > most ? prior : most);
    if (n > 0 && first < prior) {
      fine = false;
      n = 0;
    }
    if (!fine) c.refused[seq] = 1;
    units = n > 0 ? of(len, n) : 0;
    int sum = units;
    for (int d = 1; d < 64; d *= 2) {
      const int o = __shfl_up(sum, d);
      if (lane >= d) sum += o;
    }
    const bool here = units > 0 && u >= before + sum - units && u < before + sum;
    const unsigned long long found = __ballot(here);
    if (found) {
      const int src = __ffsll(found) - 1;
      unit.seq = base + src;
      unit.len = __shfl(len, src);
      unit.first = __shfl(first, src);
      unit.n = __shfl(n, src);
      unit.index = u - before - __shfl(sum - units, src);
      return true;
    }
    before += __shfl(sum, 63);
    const int last = __shfl(top, 63);
    most = last > most ? last : most;
  }
  return false;
}

// ---- append ------------------------------------------------------------------
struct AppendArgs {
  Cache c;
  const float *qkv, *rope;  // QKV rows and factors, or
  const float *k, *v;       // ready keys [rows][key heads][64] and values [rows][KV heads][64]
  const float *positions, *frequencies;  // in the factors' place: [rows][axes], [axes][n_heads][32]
  int axes;
  float *q;
  // Workgroups go to the 8 XCDs in turn. Near: those of one unit's heads, which take
  // the same factors and some the same keys, follow one another on the same one;
  // otherwise all units of four heads do.
  int near;
};

// The largest magnitude's bits in a wave, in every lane.
__device__ __forceinline__ uint32_t wave_max_bits(uint32_t v) {
  auto other = [&](auto ctrl) {
    const uint32_t o = static_cast<uint32_t>(
        __builtin_amdgcn_update_dpp(0, static_cast<int>(v), decltype(ctrl)::value, 0xf, 0xf, false));
    v = o > v ? o : v;
  };
  other(std::integral_constant<int, 0x128>());
  other(std::integral_constant<int, 0x124>());
  other(std::integral_constant<int, 0x122>());
  other(std::integral_constant<int, 0x121>());
  const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = a[0] > a[1] ? a[0] : a[1];
  const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return b[0] > b[1] ? b[0] : b[1];
}

// The value N lanes up in the 16 lanes of a DPP row (cyclically), and lane N's.
template <int N>
__device__ __forceinline__ float row_up(float v) {
  return rms_dpp<0x120 + 16 - N>(v);
}
template <int N>
__device__ __forceinline__ float row_lane(float v) {
  return rms_dpp<0x150 + N>(v);
}

// decode::norm_rope, bit for bit, of four times four rows: lane (r, c) of the wave
// holds elements 4 c .. + 3 of row 4 r + s in x[s]. The pairwise sum of squares folds
// lanes 4, 2 and 1 apart (elements 16, 8 and 4), then the lane's own (2 and 1), of both
// halves of 32; the four sums of a row's 16 lanes meet in four of them, so that the
// divisions and the root are done once for all 16 rows. A rotated pair is the lane's own.
__device__ __forceinline__ float norm_scales(const v4f (&x)[4]) {
  float sums = 0.0f;
  const int l16 = threadIdx.x & 15;
  auto total = [&](const v4f &v) {
    float p[4];
#pragma unroll
    for (int i = 0; i < 4; i++) p[i] = v[i] * v[i];
#pragma unroll
    for (int i = 0; i < 4; i++) p[i] = p[i] + row_up<4>(p[i]);
#pragma unroll
    for (int i = 0; i < 4; i++) p[i] = p[i] + row_up<2>(p[i]);
#pragma unroll
    for (int i = 0; i < 4; i++) p[i] = p[i] + row_up<1>(p[i]);
    const float leaf = (p[0] + p[2]) + (p[1] + p[3]);
    return row_lane<0>(leaf) + row_lane<8>(leaf);
  };
#pragma unroll
  for (int s = 0; s < 4; s++) {
    const float t = total(x[s]);
    sums = l16 == s ? t : sums;
  }
  return __fdiv_rn(1.0f, __builtin_sqrtf(__fdiv_rn(sums, 64.0f) + 1.1920929e-7f));
}
// Of row s: lane s of the 16 has it.
__device__ __forceinline__ float norm_scale(float scales, int s) {
  return s == 0 ? row_lane<0>(scales) : s == 1 ? row_lane<1>(scales) : s == 2 ? row_lane<2>(scales) : row_lane<3>(scales);
}
__device__ __forceinline__ v4f rotated(const v4f &x, float scale, const v4f &f) {
  const v4f y = {x[0] * scale, x[1] * scale, x[2] * scale, x[3] * scale};
  return v4f{y[0] * f[0] - y[1] * f[1], y[0] * f[1] + y[1] * f[0], y[2] * f[2] - y[3] * f[3], y[2] * f[3] + y[3] * f[2]};
}
__device__ __forceinline__ void norm_rotate(v4f (&x)[4], const v4f (&f)[4]) {
  const float scales = norm_scales(x);
#pragma unroll
  for (int s = 0; s < 4; s++) x[s] = rotated(x[s], norm_scale(scales, s), f[s]);
}

// Units of an append: the blocks of a sequence's rows, the first and the last two
// together (they read and write the FP32 blocks), the others one by one.
__device__ __forceinline__ int touched(int len, int n) { return (len + n - 1) / kBlock - len / kBlock + 1; }

// Four bytes of four words to four words of four bytes.
__device__ __forceinline__ void turn_bytes(uint32_t (&w)[4]) {
  const uint32_t a01 = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u), a23 = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u);
  const uint32_t b01 = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u), b23 = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
  w[0] = __builtin_amdgcn_perm(a23, a01, 0x05040100u);
  w[1] = __builtin_amdgcn_perm(a23, a01, 0x07060302u);
  w[2] = __builtin_amdgcn_perm(b23, b01, 0x05040100u);
  w[3] = __builtin_amdgcn_perm(b23, b01, 0x07060302u);
}

// Writes a block of a stored head: `x` holds its positions, those before the unit's rows
// from the FP32 block `open` (row0 < 0) if that is still the block's.
__device__ __forceinline__ void put_block(const Cache &c, const Unit &unit, bool is_key, int held, int at_head, size_t slot, int block,
                                          int last_block, v4f (&x)[4]) {
  const int lane = threadIdx.x & 63, r4 = lane / 16 * 4, e4 = lane % 16 * 4;
  const int row0 = block * kBlock - unit.len;
  float *const open = c.open + (slot + block % 2) * kBlock * 64;
  const bool earlier = row0 < 0;
  const long number = c.block_at(unit.seq, block, held, at_head);
  if (number < 0) {
    c.refused[unit.seq] = 1;
    return;
  }
  int8_t *const codes = (is_key ? c.k_codes : c.v_codes) + number * kBlockBytes;
  float *const scale_at = (is_key ? c.k_scales : c.v_scales) + number;
  int32_t *const writer_at = (is_key ? c.k_writers : c.v_writers) + number;
  const bool kept = earlier && c.tags[slot + block % 2] == block && *writer_at == unit.seq;
  if (earlier && !kept) {
    // From the codes.
    const float scale = *scale_at;
    uint32_t w[4];
#pragma unroll
    for (int s = 0; s < 4; s++)
      w[s] = *reinterpret_cast<const uint32_t *>(is_key ? codes + s * 256 + lane * 4 : codes + (e4 + s) * kBlock + r4);
    if (!is_key) turn_bytes(w);
#pragma unroll
    for (int s = 0; s < 4; s++)
      if (row0 + r4 + s < 0)
        x[s] = v4f{sdwa_cvt<0>(w[s]) * scale, sdwa_cvt<1>(w[s]) * scale, sdwa_cvt<2>(w[s]) * scale, sdwa_cvt<3>(w[s]) * scale};
  }
  uint32_t big = 0;
#pragma unroll
  for (int s = 0; s < 4; s++) {
    if (row0 + r4 + s >= unit.n) x[s] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint32_t bits = __float_as_uint(x[s][i]) & 0x7fffffffu;
      big = bits > big ? bits : big;
    }
  }
  big = wave_max_bits(big);
  float scale = __fdiv_rn(__uint_as_float(big), 127.0f);
  if (scale < 1.17549435e-38f) scale = 0.0f;
  float inverse = scale > 0.0f ? __fdiv_rn(1.0f, scale) : 0.0f;
  if (big >= 0x7f800000u) {
    scale = __builtin_nanf("");
    inverse = 0.0f;
  }
  uint32_t w[4];
#pragma unroll
  for (int s = 0; s < 4; s++) {
    // 1.5 2^23 + code, rounded to nearest even, holds the code in its low byte.
    uint32_t bits[4];
#pragma unroll
    for (int i = 0; i < 4; i++) bits[i] = __float_as_uint(x[s][i] * inverse + 12582912.0f);
    const uint32_t lo = __builtin_amdgcn_perm(bits[1], bits[0], 0x0c0c0400u);
    w[s] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(bits[3], bits[2], 0x0c0c0400u), lo, 0x05040100u);
  }
  if (!is_key) turn_bytes(w);
#pragma unroll
  for (int s = 0; s < 4; s++)
    *reinterpret_cast<uint32_t *>(is_key ? codes + s * 256 + lane * 4 : codes + (e4 + s) * kBlock + r4) = w[s];
  if (lane == 0) {
    *scale_at = scale;
    *writer_at = unit.seq;
  }
  if (block >= last_block - 1) {
#pragma unroll
    for (int s = 0; s < 4; s++) {
      const int row = row0 + r4 + s;
      if (row < unit.n && (row >= 0 || !kept)) *reinterpret_cast<v4f *>(open + (r4 + s) * 64 + e4) = x[s];
    }
    if (lane == 0) c.tags[slot + block % 2] = block;
  }
}

// A wave takes one unit and one head: a stored head (keys, then values), or with QKV
// a query head. Lane (r, c): elements 4 c .. + 3 of the block's positions 4 r + s, s =
// 0 .. 3, so that a load or store of FP32 rows is 1 KB, key codes go to memory as
// they stand (256 bytes for each s) and a dim's codes of four positions are one word.
// Bound: the rows and factors read, the queries written. 15,243 rows of four prompts
// (16 query and key heads, 8 value heads) take 62 us for 188 MB read and 87 written,
// 4.4 TB/s where a copy reaches 5.1; a row of each of 64 sequences 6.4 us, which is
// the launch and three dependent trips to memory (batch, table, rows).
template <bool QKV>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
  const Cache &c = a.c;
  const int lane = threadIdx.x & 63, r4 = lane / 16 * 4, e4 = lane % 16 * 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int at_unit = a.near ? (blockIdx.z * gridDim.y + blockIdx.y) * 8 + blockIdx.x % 8 : blockIdx.x;
  const int head = (a.near ? blockIdx.x / 8 : blockIdx.y) * 4 + wave, stored = c.key_heads + c.kv_heads;
  const auto of = [](int len, int n) {
    const int blocks = touched(len, n);
    return blocks <= 3 ? 1 : blocks - 2;
  };
  Unit unit;
  const bool found = find_unit(c, at_unit, of, unit);
  if (at_unit == 0 && head == 0 && c.row_start) {
    // Marks every refused sequence.
    Unit none;
    find_unit(c, 0x7fffffff, of, none);
  }
  if (!found || head >= stored + (QKV ? c.n_heads : 0)) return;
  const bool is_key = head < c.key_heads, is_query = head >= stored;
  // Where the head stands in a row, and whose factors its pairs take.
  const float *source;
  size_t width;
  int pair = 0;
  if constexpr (QKV) {
    width = static_cast<size_t>(c.n_heads + 2 * c.kv_heads) * 64;
    int from;
    if (is_query) {
      from = pair = head - stored;
    } else if (is_key) {
      from = c.n_heads + head * c.kv_heads / c.key_heads;
      pair = head * (c.n_heads / c.key_heads);
    } else {
      from = c.n_heads + c.kv_heads + head - c.key_heads;
    }
    source = a.qkv + from * 64;
  } else {
    width = static_cast<size_t>(is_key ? c.key_heads : c.kv_heads) * 64;
    source = (is_key ? a.k : a.v) + (is_key ? head : head - c.key_heads) * 64;
  }
  const bool turned = QKV && (is_key || is_query);
  const int first_block = unit.len / kBlock, blocks = touched(unit.len, unit.n), last_block = first_block + blocks - 1;
  const int held = is_key ? c.key_heads : c.kv_heads, at_head = is_key ? head : head - c.key_heads;
  const size_t slot = (static_cast<size_t>(unit.seq) * stored + head) * 2;

  auto process = [&](int block) {
    const int row0 = block * kBlock - unit.len;  // the row of its first position
    float *const open = is_query ? nullptr : c.open + (slot + block % 2) * kBlock * 64;
    const bool earlier = !is_query && row0 < 0;
    // Earlier positions from the FP32 block, new ones from the rows.
    v4f x[4], f[4];
#pragma unroll
    for (int s = 0; s < 4; s++) {
      const int row = row0 + r4 + s;
      const size_t at = unit.first + (row < 0 ? 0 : row < unit.n ? row : unit.n - 1);
      const float *from = earlier && row < 0 ? open + (r4 + s) * 64 : source + at * width;
      x[s] = *reinterpret_cast<const v4f *>(from + e4);
      if (turned) f[s] = *reinterpret_cast<const v4f *>(a.rope + (at * c.n_heads + pair) * 64 + e4);
    }
    if (turned) {
      v4f y[4] = {x[0], x[1], x[2], x[3]};
      norm_rotate(y, f);
      if (is_query) {
#pragma unroll
        for (int s = 0; s < 4; s++) {
          const int row = row0 + r4 + s;
          if (row >= 0 && row < unit.n)
            *reinterpret_cast<v4f *>(a.q + (static_cast<size_t>(unit.first + row) * c.n_heads + pair) * 64 + e4) = y[s];
        }
        return;
      }
#pragma unroll
      for (int s = 0; s < 4; s++)
        if (row0 + r4 + s >= 0) x[s] = y[s];
    }
    put_block(c, unit, is_key, held, at_head, slot, block, last_block, x);
  };
  if (unit.index > 0) {
    process(first_block + unit.index);
    return;
  }
  process(first_block);
  // The last two, which may be written where the first was read.
  for (int block = last_block - 1 > first_block ? last_block - 1 : first_block + 1; block <= last_block; block++)
    process(block);
}

// The row step from positions (rotary.hpp): a wave takes one unit and one query head, and with
// it the key head that is turned by the same factors, or one value head. Lanes are as
// in append_kernel; a lane forms the factors of its two pairs in its four rows, bitwise
// those of focr_rotary_factors, while the rows are on their way. Bound: for prompts the vector
// instructions, some 1,400 for a block and a head, 350 of them the factors', and the trips to
// memory that five waves on a SIMD leave uncovered: 15,243 rows of four with three axes
// take 55 to 61 us (3.3 to 3.7 TB/s); for single rows trips one after another, 64 sequences
// 7.9 us.
template <int AXES>
__global__ __launch_bounds__(256, 5) void turn_kernel(AppendArgs a) {
  const Cache &c = a.c;
  const int lane = threadIdx.x & 63, r4 = lane / 16 * 4, e4 = lane % 16 * 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int at_unit = a.near ? (blockIdx.z * gridDim.y + blockIdx.y) * 8 + blockIdx.x % 8 : blockIdx.x;
  const int task = (a.near ? blockIdx.x / 8 : blockIdx.y) * 4 + wave;
  const auto of = [](int len, int n) {
    const int blocks = touched(len, n);
    return blocks <= 3 ? 1 : blocks - 2;
  };
  Unit unit;
  const bool found = find_unit(c, at_unit, of, unit);
  if (at_unit == 0 && task == 0 && c.row_start) {
    // Marks every refused sequence.
    Unit none;
    find_unit(c, 0x7fffffff, of, none);
  }
  if (!found || task >= c.n_heads + c.kv_heads) return;
  const bool is_value = task >= c.n_heads;
  const int query = task, repeat = c.n_heads / c.key_heads, value_head = task - c.n_heads;
  const bool has_key = !is_value && query % repeat == 0;
  const int key_head = query / repeat;
  const size_t width = static_cast<size_t>(c.n_heads + 2 * c.kv_heads) * 64;
  const int stored = c.key_heads + c.kv_heads, at_stored = is_value ? c.key_heads + value_head : key_head;
  const size_t slot = (static_cast<size_t>(unit.seq) * stored + at_stored) * 2;
  const float *const key_source = a.qkv + (is_value ? c.n_heads + c.kv_heads + value_head : c.n_heads + key_head * c.kv_heads / c.key_heads) * 64;
  const int first_block = unit.len / kBlock, blocks = touched(unit.len, unit.n), last_block = first_block + blocks - 1;
  __shared__ float places[4][kBlock * kMaxAxes];  // a wave's: positions of its block's rows
  __shared__ float2 speeds[4][AXES][16];  // and the frequencies of its pairs
  if (!is_value)
#pragma unroll
    for (int x = 0; x < AXES; x++)
      speeds[wave][x][e4 / 4] = *reinterpret_cast<const float2 *>(a.frequencies + (static_cast<size_t>(x) * c.n_heads + query) * 32 + e4 / 2);

  auto process = [&](int block) {
    const int row0 = block * kBlock - unit.len;  // the row of its first position
    const float *const open = c.open + (slot + block % 2) * kBlock * 64;
    v4f x[4], y[4];
    float place = 0.0f;
    if (!is_value && lane < kBlock * AXES) {
      const int row = row0 + lane / AXES;
      place = a.positions[(unit.first + static_cast<size_t>(row < 0 ? 0 : row < unit.n ? row : unit.n - 1)) * AXES + lane % AXES];
    }
#pragma unroll
    for (int s = 0; s < 4; s++) {
      const int row = row0 + r4 + s;
      const size_t at = unit.first + (row < 0 ? 0 : row < unit.n ? row : unit.n - 1);
      // Earlier positions from the FP32 block, new ones from the rows.
      if (is_value || has_key) x[s] = *reinterpret_cast<const v4f *>((row < 0 ? open + (r4 + s) * 64 : key_source + at * width) + e4);
      if (!is_value) y[s] = *reinterpret_cast<const v4f *>(a.qkv + query * 64 + at * width + e4);
    }
    if (!is_value) {
      places[wave][lane] = place;
      // One pair of one row after another, positions and frequencies from LDS, so that few
      // 64-bit numbers are held: all at once, at 115 registers, four waves fit on a SIMD and
      // the same prompts take 66 us; bounded to 80 registers, which spill, 78.
      const float scales = norm_scales(y);
      float key_scales = 0.0f;
      if (has_key) key_scales = norm_scales(x);
#pragma unroll
      for (int s = 0; s < 4; s++) {
        // A step of few rows leaves most places of a block without one.
        const int row = row0 + r4 + s;
        if (unit.n < kBlock && !__any(row >= 0 && row < unit.n)) continue;
        __builtin_amdgcn_sched_barrier(0);
        v4f f;
#pragma unroll
        for (int j = 0; j < 2; j++) {
          double angle;
#pragma unroll
          for (int i = 0; i < AXES; i++) {
            const double at = places[wave][(r4 + s) * AXES + i], speed = j == 0 ? speeds[wave][i][e4 / 4].x : speeds[wave][i][e4 / 4].y;
            angle = i == 0 ? at * speed : __builtin_fma(at, speed, angle);
          }
          const float2 turn = cos_sin(angle);
          f[2 * j] = turn.x;
          f[2 * j + 1] = turn.y;
          __builtin_amdgcn_sched_barrier(0);
        }
        asm volatile("" ::: "memory");  // read again for the next row, not held
        const v4f turned = rotated(y[s], norm_scale(scales, s), f);
        if (row >= 0 && row < unit.n)
          *reinterpret_cast<v4f *>(a.q + (static_cast<size_t>(unit.first + row) * c.n_heads + query) * 64 + e4) = turned;
        if (has_key) {
          const v4f key = rotated(x[s], norm_scale(key_scales, s), f);
          if (row >= 0) x[s] = key;
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      if (!has_key) return;
    }
    put_block(c, unit, !is_value, is_value ? c.kv_heads : c.key_heads, is_value ? value_head : key_head, slot, block, last_block, x);
  };
  // The first, or one of a long unit's, and with the first the last two, which may be
  // written where the first was read.
  int block = first_block + unit.index;
  const int end = unit.index > 0 ? block : last_block;
  while (true) {
    process(block);
    if (block >= end) break;
    block = block + 1 > last_block - 1 ? block + 1 : last_block - 1;
  }
}

// ---- reading back --------------------------------------------------------------
// A wave takes one block of a sequence's rows and one stored head. Bound by the FP32
// rows written: 15,243 rows of 24 heads take 25 us (118 MB moved, 4.7 TB/s).
__global__ __launch_bounds__(256) void read_kernel(Cache c, float *__restrict__ k, float *__restrict__ v) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int head = blockIdx.y * 4 + wave, stored = c.key_heads + c.kv_heads;
  const auto of = [](int len, int n) { return touched(len, n); };
  Unit unit;
  const bool found = find_unit(c, blockIdx.x, of, unit);
  if (blockIdx.x == 0 && head == 0 && c.row_start) {
    Unit none;
    find_unit(c, 0x7fffffff, of, none);
  }
  if (!found || head >= stored) return;
  const bool is_key = head < c.key_heads;
  const int held = is_key ? c.key_heads : c.kv_heads, at_head = is_key ? head : head - c.key_heads;
  const int block = unit.len / kBlock + unit.index, row0 = block * kBlock - unit.len;
  const long number = c.block_at(unit.seq, block, held, at_head);
  if (number < 0) c.refused[unit.seq] = 1;
  const size_t at = number < 0 ? 0 : number;
  const float scale = number < 0 ? __builtin_nanf("") : (is_key ? c.k_scales : c.v_scales)[at];
  // Lane (r, c): elements 4 c .. + 3 of positions 4 r + s, as they were appended.
  const int r4 = lane / 16 * 4, e4 = lane % 16 * 4;
  const int8_t *const codes = (is_key ? c.k_codes : c.v_codes) + at * kBlockBytes;
  float *const to = (is_key ? k : v) + at_head * 64 + e4;
  uint32_t w[4];
#pragma unroll
  for (int s = 0; s < 4; s++)
    w[s] = *reinterpret_cast<const uint32_t *>(is_key ? codes + s * 256 + lane * 4 : codes + (e4 + s) * kBlock + r4);
  if (!is_key) turn_bytes(w);
#pragma unroll
  for (int s = 0; s < 4; s++) {
    const int row = row0 + r4 + s;
    if (row >= 0 && row < unit.n)
      *reinterpret_cast<v4f *>(to + static_cast<size_t>(unit.first + row) * held * 64) =
          v4f{sdwa_cvt<0>(w[s]) * scale, sdwa_cvt<1>(w[s]) * scale, sdwa_cvt<2>(w[s]) * scale, sdwa_cvt<3>(w[s]) * scale};
  }
}

// ---- attention -----------------------------------------------------------------
struct AttendArgs {
  Cache c;
  const float *q, *sinks;
  float *out;
  float *part_o, *part_md;  // [row][head][part][64], [..][2]
  int max_len, chunk, parts, tiles;  // tiles: of 16 columns, for as many rows as a sequence can have
};
// Over a shared prefix: positions below base are those of sequence `prefix`, in the first
// first_part of the parts; own_parts hold a sequence's own.
struct SharedArgs : AttendArgs {
  int own_parts, first_part, base, prefix, prefix_chunk, prefix_tiles, prefix_blocks, beside;
  int alone;  // a sequence's own by waves
};
template <typename Args>
constexpr bool kShared = std::is_same<Args, SharedArgs>::value;

// A sequence's rows for attention; false where there is nothing to do (n = 0) or it
// is refused (bad), but for what `overlaps` says.
template <typename Args>
__device__ __forceinline__ bool attend_span(const Args &a, int seq, int &len, int &first, int &n, bool &bad) {
  bad = !a.c.span(seq, len, first, n);
  if (n > 8 || (n > 0 && len + n > a.max_len)) bad = true;
  if constexpr (kShared<Args>)
    if (n > 0 && len < a.base) bad = true;
  return n > 0 && !bad;
}

// Whether a sequence's rows, from `first` on, begin before those of a sequence before it
// end, as find_unit refuses them. A wave's question. Starts that do not decrease never
// do, so mostly these are all that is looked at: each lane's of the first 64 (`start_of`,
// loaded ahead of the question), and of 256 at a time.
__device__ __forceinline__ int start_of(const Cache &c, int seq) {
  const int at = 1 + static_cast<int>(threadIdx.x & 63);
  return c.row_start ? c.row_start[at < seq ? at : seq] : 0;
}
__device__ __forceinline__ bool overlaps(const Cache &c, int seq, int first, int start) {
  if (!c.row_start) return false;
  const int lane = threadIdx.x & 63;
  int top = start;
  for (int base = 65; base < seq; base += 256) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int at = base + 64 * i + lane, other = c.row_start[at < seq ? at : seq];
      top = other > top ? other : top;
    }
  }
  if (!__any(top > first)) return false;
  bool found = false;
  for (int base = 0; base < seq; base += 64) {
    int len, other, n;
    const int at = base + lane;
    if (at < seq && c.span(at, len, other, n) && n > 0 && other + n > first) found = true;
  }
  return __any(found);
}

// out = o / den / (1 + exp(sink - lse)), lse = (m + log2(den)) ln 2.
__device__ __forceinline__ float sink_factor(const float *sinks, int head, float m, float den) {
  if (!sinks) return 1.0f;
  const float lse = (m + log2f(den)) * 0.693147180559945f;
  return __fdiv_rn(1.0f, 1.0f + expf_acc(sinks[head] - lse));
}

constexpr int kMaxParts = 256;

// The weight of a softmax state among states whose largest maximum is `top`. A state
// without a maximum holds no key that its row sees (weight 0), or only NaN (its sum).
__device__ __forceinline__ float state_weight(float m, float den, float top) {
  if (m == -__builtin_inff()) return den != den ? den : 0.0f;
  return __builtin_amdgcn_exp2f(m - top);
}

// The rows of a refused sequence, where they are rows of the call: NaN. Only those that
// can be no other sequence's: behind all starts before its own and before all later ones.
__device__ __forceinline__ void refuse_rows(const AttendArgs &a, int seq, int head0, int heads) {
  const Cache &c = a.c;
  const int lane = threadIdx.x & 63;
  const int begin = c.row_start ? c.row_start[seq] : seq, end = c.row_start ? c.row_start[seq + 1] : seq + 1;
  if (lane == 0) c.refused[seq] = 1;
  if (begin < 0 || end > c.rows) return;
  int from = begin, to = end;
  if (c.row_start) {
    for (int at = lane; at <= c.n_seqs; at += 64) {
      const int start = c.row_start[at];
      if (at <= seq)
        from = start > from ? start : from;
      else
        to = start < to ? start : to;
    }
    for (int d = 1; d < 64; d *= 2) {
      const int f = __shfl_xor(from, d), t = __shfl_xor(to, d);
      from = f > from ? f : from;
      to = t < to ? t : to;
    }
  }
  for (int row = from; row < to; row++)
    for (int h = head0; h < head0 + heads; h++)
      a.out[(static_cast<size_t>(row) * c.n_heads + h) * 64 + lane] = __builtin_nanf("");
}

// Largest and sum of the 16 lanes of a DPP row, in each of them.
template <int N>
__device__ __forceinline__ float row_ror(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x120 + N, 0xf, 0xf, false));
}
__device__ __forceinline__ float row_max(float v) {
  v = __builtin_fmaxf(v, row_ror<8>(v));
  v = __builtin_fmaxf(v, row_ror<4>(v));
  v = __builtin_fmaxf(v, row_ror<2>(v));
  return __builtin_fmaxf(v, row_ror<1>(v));
}

// A column's state from those of its runs, [run][column] in LDS: four dims of it.
__device__ __forceinline__ v4f join_runs(const float *s_m, const float *s_den, const float (*s_o)[68], int col, int wide,
                                         int runs, int dim, float &top, float &total) {
  top = s_m[col];
  total = 0.0f;
  for (int w = 1; w < runs; w++) top = __builtin_fmaxf(top, s_m[w * wide + col]);
  v4f o = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int w = 0; w < runs; w++) {
    const int at = w * wide + col;
    const float f = state_weight(s_m[at], s_den[at], top);
    total = fmaf_(s_den[at], f, total);
    const v4f x = *reinterpret_cast<const v4f *>(&s_o[at][dim]);
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] = fmaf_(x[i], f, o[i]);
  }
  return o;
}
__device__ __forceinline__ void store_part(const AttendArgs &a, size_t at, int dim, const v4f &o, float top, float total) {
  *reinterpret_cast<v4f *>(a.part_o + at * 64 + dim) = o;
  if (dim == 0) *reinterpret_cast<float2 *>(a.part_md + at * 2) = make_float2(top, total);
}

// A workgroup takes one sequence, one key head's queries (its query heads times the
// sequence's rows: columns, up to 16 of them) and one part of the keys. A wave takes
// four columns and one run of the part's keys, 64 (four blocks) at a time: up to four
// columns leave each wave a run of its own, up to eight two waves, more all four.
//
// Scores. A query row is integers i 2^(e - 30) of four signed bytes (2^e above its
// largest element, so to 2^-30 of it: elements down to 2^-6 of it keep all their
// bits). Row 4 q + d of the INT8 matrix product holds byte d of query q, column j of
// key tile t is key 4 j + t as its codes stand: lane (j, q) gets the four exact sums of
// its four keys with its query, and nothing is computed twice. Weights. w = exp2(s - m)
// times the block's value scale in FP32, over the power of two above the largest such
// scale so far and times 2^64 (so that weights 2^-174 below that keep all their bits),
// is the sum of three BF16 numbers, its own bits eight at a time: part d of query q is
// column 4 d + q of the second product, whose operands are the value codes as BF16
// numbers (exact) and these parts, turned through LDS. So every product is exact,
// whatever the magnitudes of the other keys' weights and values, and sums round as
// FP32's do; integers of one step for a run's weights would lose those far below the
// largest. The sums stay in the accumulators, which are scaled when m or the power of
// two changes.
//
// Bound: the codes, read once. 64 sequences of up to 8,192 positions (346,572 in all,
// 16 key and 8 value heads) take 107 us, 623 MB from memory at 5.8 TB/s; 535 MB
// are needed, as two key heads' workgroups do not read all of their values together
// (both in one workgroup: 549 MB, but 8 % longer, as fewer bytes are on their way). One
// sequence of 131,072 takes 25 us (137 MB, 5.6 TB/s) and its merge 5; 101
// positions take 5.7 us, the launch and four dependent trips to memory.
struct Stage {
  v4i k[4], v[4];
  float k_scale, v_scale;
  bool none;
};
struct Found {
  int k_page, v_page;
};

// 64 keys: lane's key block is l16 / 4 of four, its value block g. In a page of 64
// positions or more (WIDE) they follow one another, and their addresses are scalar
// but for the lane's share; otherwise each lane looks its blocks' pages up (past the
// last block, that one again). A block without a page is NaN.
template <bool WIDE>
struct Reader {
  typedef __attribute__((address_space(4))) const int32_t scalar_table;  // read by scalar loads
  const Cache &c;
  const int32_t *table;
  int key_head, value_head, last_block;
  bool missing = false;

  __device__ __forceinline__ Reader(const Cache &cache, int seq, int head, int limit)
      : c(cache), table(cache.table + static_cast<size_t>(seq) * cache.seq_pages), key_head(head),
        value_head(head * cache.kv_heads / cache.key_heads), last_block((limit - 1) / kBlock) {}

  __device__ __forceinline__ Found find(int key0) const {
    const int l16 = threadIdx.x & 15, g = threadIdx.x >> 4 & 3;
    Found f;
    const int b = key0 / kBlock;
    if constexpr (WIDE) {
      const int at = b < last_block ? b : last_block;
      f.k_page = f.v_page = reinterpret_cast<scalar_table *>(reinterpret_cast<uintptr_t>(table))[at >> c.shift];
    } else {
      f.k_page = table[(b + l16 / 4 < last_block ? b + l16 / 4 : last_block) >> c.shift];
      f.v_page = table[(b + g < last_block ? b + g : last_block) >> c.shift];
    }
    return f;
  }
  __device__ __forceinline__ void load(const Found &f, int key0, Stage &s) {
    const int l16 = threadIdx.x & 15, g = threadIdx.x >> 4 & 3, blocks_mask = (1 << c.shift) - 1;
    const int k_lane = l16 % 4 * 64 + g * 16, v_lane = l16 * 16;
    const int b = key0 / kBlock;
    const bool none = f.k_page < 0;
    missing |= none;
    const long kp = none ? 0 : f.k_page, vp = f.v_page < 0 ? 0 : f.v_page;
    if constexpr (WIDE) {
      const long kn = ((kp * c.key_heads + key_head) << c.shift) + (b & blocks_mask);
      const long vn = ((kp * c.kv_heads + value_head) << c.shift) + (b & blocks_mask);
      const int8_t *k = c.k_codes + kn * kBlockBytes, *v = c.v_codes + vn * kBlockBytes;
      s.k_scale = (c.k_scales + kn)[l16 / 4];
      s.v_scale = (c.v_scales + vn)[l16 / 4];
      s.none = none;
#pragma unroll
      for (int t = 0; t < 4; t++) s.k[t] = *reinterpret_cast<const v4i *>(k + t * 256 + (l16 / 4 * kBlockBytes + k_lane));
#pragma unroll
      for (int d = 0; d < 4; d++) s.v[d] = *reinterpret_cast<const v4i *>(v + d * 256 + (g * kBlockBytes + v_lane));
    } else {
      const int k_in = (b + l16 / 4 < last_block ? b + l16 / 4 : last_block) & blocks_mask;
      const int v_in = (b + g < last_block ? b + g : last_block) & blocks_mask;
      const long kn = ((kp * c.key_heads + key_head) << c.shift) + k_in;
      const long sn = ((kp * c.kv_heads + value_head) << c.shift) + k_in;
      const long vn = ((vp * c.kv_heads + value_head) << c.shift) + v_in;
      s.k_scale = c.k_scales[kn];
      s.v_scale = c.v_scales[sn];
      s.none = none;
      const int8_t *k = c.k_codes + kn * kBlockBytes + k_lane, *v = c.v_codes + vn * kBlockBytes + v_lane;
#pragma unroll
      for (int t = 0; t < 4; t++) s.k[t] = *reinterpret_cast<const v4i *>(k + t * 256);
#pragma unroll
      for (int d = 0; d < 4; d++) s.v[d] = *reinterpret_cast<const v4i *>(v + d * 256);
    }
  }
};

// Four columns of a wave. Lane l16 holds row l16 of the first product (query l16 / 4,
// byte l16 % 4), lane (l16, g) works on query g.
struct Quad {
  v4i digit;
  float factor, m, den;
  int visible;  // keys that query g sees
  v4f acc[4];

  // From 16 elements of query l16 / 4 (lane (l16, g): 16 g .. + 15).
  __device__ __forceinline__ void begin(const float4 (&x)[4]) {
    const int l16 = threadIdx.x & 15, g = threadIdx.x >> 4 & 3;
    uint32_t big = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float y[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const uint32_t bits = __float_as_uint(y[j]) & 0x7fffffffu;
        big = bits > big ? bits : big;
      }
    }
    auto p = __builtin_amdgcn_permlane16_swap(big, big, false, false);
    big = p[0] > p[1] ? p[0] : p[1];
    p = __builtin_amdgcn_permlane32_swap(big, big, false, false);
    big = p[0] > p[1] ? p[0] : p[1];
    const bool finite = big < 0x7f800000u;
    int e = !finite || big == 0 ? 0 : __builtin_amdgcn_frexp_expf(__uint_as_float(big));
    e = e < -90 ? -90 : e;
    // log2(e) / 8: scores in powers of two. From query l16 / 4 to query g.
    const float scale = finite ? __builtin_ldexpf(0.180336880111120426f, e - 30) : __builtin_nanf("");
    factor = __int_as_float(__builtin_amdgcn_ds_bpermute(4 * (4 * g), __float_as_int(scale)));
    // Adding 128 to each lower byte of i and inverting their top bits leaves signed
    // bytes whose weighted sum is i.
    auto bytes = [&](float f) {
      const int i = finite ? static_cast<int>(__builtin_rintf(__builtin_ldexpf(f, 30 - e))) : 0;
      return (static_cast<uint32_t>(i) + 0x00808080u) ^ 0x00808080u;
    };
    // Byte l16 % 4 of four values.
    const uint32_t pick = 0x0c0c0400u + 0x0101u * (l16 % 4);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint32_t lo = __builtin_amdgcn_perm(bytes(x[i].y), bytes(x[i].x), pick);
      const uint32_t hi = __builtin_amdgcn_perm(bytes(x[i].w), bytes(x[i].z), pick);
      digit[i] = static_cast<int>(lo | hi << 16);
    }
    m = -__builtin_inff();
    den = 0.0f;
#pragma unroll
    for (int d = 0; d < 4; d++) acc[d] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  }

  // The sums times `scaled` of query g: column 4 d + q's lanes take that of query q.
  __device__ __forceinline__ void rescale(float scaled) {
    const int l16 = threadIdx.x & 15;
    const float s0 = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(scaled), 0));
    const float s1 = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(scaled), 16));
    const float s2 = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(scaled), 32));
    const float s3 = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(scaled), 48));
    const float f = l16 & 2 ? (l16 & 1 ? s3 : s2) : (l16 & 1 ? s1 : s0);
#pragma unroll
    for (int d = 0; d < 4; d++)
#pragma unroll
      for (int i = 0; i < 4; i++) acc[d][i] = acc[d][i] * f;
  }

  // The run's state to LDS: the four columns' m and den, and their sums [column][68].
  __device__ __forceinline__ void end(int power, float *to_m, float *to_den, float (*to_o)[68]) {
    const int l16 = threadIdx.x & 15, g = threadIdx.x >> 4 & 3;
    den = den + row_ror<8>(den);
    den = den + row_ror<4>(den);
    den = den + row_ror<2>(den);
    den = den + row_ror<1>(den);
    if (l16 == 0) {
      to_m[g] = m;
      to_den[g] = den;
    }
#pragma unroll
    for (int d = 0; d < 4; d++) {
      v4f o;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        // Lane l16 < 4: the sums of lanes l16, + 4, + 8, the upper part's first.
        const float x = acc[d][i];
        o[i] = __builtin_ldexpf((row_ror<8>(x) + row_ror<12>(x)) + x, power - 64);
      }
      if (l16 < 4) *reinterpret_cast<v4f *>(&to_o[l16][16 * d + 4 * g]) = o;
    }
  }
};

// Two FP32 numbers' upper halves, the first one's low.
__device__ __forceinline__ uint32_t upper(uint32_t second, uint32_t first) {
  return __builtin_amdgcn_perm(second, first, 0x07060302u);
}
// Eight codes as BF16 numbers.
__device__ __forceinline__ v8bf codes_of(int first, int second) {
  const uint32_t w[2] = {static_cast<uint32_t>(first), static_cast<uint32_t>(second)};
  v4i to;
#pragma unroll
  for (int i = 0; i < 2; i++) {
    to[2 * i] = static_cast<int>(upper(__float_as_uint(sdwa_cvt<1>(w[i])), __float_as_uint(sdwa_cvt<0>(w[i]))));
    to[2 * i + 1] = static_cast<int>(upper(__float_as_uint(sdwa_cvt<3>(w[i])), __float_as_uint(sdwa_cvt<2>(w[i]))));
  }
  return __builtin_bit_cast(v8bf, to);
}

// The parts of the weights: [column 4 d + q][64 keys], a wave's own for four columns.
// Rows of 72, so that 16 columns' 16 bytes lie in different banks; there is no fourth part.
constexpr int kTurned = 72;

// 64 keys from key0 on for a wave's four columns. `turned` is the wave's own. 2^power
// is above every block scale of the values so far.
__device__ __forceinline__ void consume(Quad &u, int &power, const Stage &s, int key0, int last_block, uint16_t *turned) {
  const int l16 = threadIdx.x & 15, g = threadIdx.x >> 4 & 3;
  const float ninf = -__builtin_inff();
  // Blocks that hold none of the sequence's positions do not count; NaN reaches a
  // row by its scores, which are those of the keys it sees.
  float v_scale = key0 / kBlock + l16 / 4 <= last_block ? s.v_scale : 0.0f;
  const bool bad = v_scale != v_scale;
  const float k_scale = s.none || bad ? __builtin_nanf("") : s.k_scale;
  v_scale = bad ? 0.0f : v_scale;
  // The largest value scale of the four blocks (lanes 4 b .. + 3 of a row).
  float widest = __builtin_fmaxf(v_scale, row_ror<4>(v_scale));
  widest = __builtin_fmaxf(widest, row_ror<8>(widest));
  int above = widest > 0.0f ? __builtin_amdgcn_frexp_expf(widest) : -300;
  above = __builtin_amdgcn_readfirstlane(above > power ? above : power);
  const int lower = power - above;
  power = above;
  const float weight = __builtin_ldexpf(v_scale, 64 - power);
  uint16_t *const turn_to = turned + g * kTurned + 4 * l16;
  const uint16_t *const turn_from = turned + l16 * kTurned + 16 * g;
  float p[4];
  const float factor = u.factor * k_scale;
#pragma unroll
  for (int t = 0; t < 4; t++) {
    const v4i zero = {0, 0, 0, 0};
    const v4i dots = __builtin_amdgcn_mfma_i32_16x16x64_i8(u.digit, s.k[t], zero, 0, 0, 0);
    // A sum is below 2^20, so two of them fit 32 bits.
    const float sum = fmaf_(static_cast<float>((dots[3] << 8) + dots[2]), 65536.0f, static_cast<float>((dots[1] << 8) + dots[0]));
    p[t] = sum * factor;
    if (key0 + 4 * l16 + t >= u.visible) p[t] = ninf;
  }
  float top = __builtin_fmaxf(__builtin_fmaxf(p[0], p[1]), __builtin_fmaxf(p[2], p[3]));
  top = __builtin_fmaxf(u.m, row_max(top));
  const float from = top == ninf ? 0.0f : top;
  if (__any(top > u.m) || lower < 0) {
    const float keep = __builtin_amdgcn_exp2f(u.m - from);
    u.den = u.den * keep;
    u.rescale(__builtin_ldexpf(keep, lower));
    u.m = top;
  }
  uint32_t part[3][4];
#pragma unroll
  for (int t = 0; t < 4; t++) {
    const float e = __builtin_amdgcn_exp2f(p[t] - from);
    u.den = u.den + e;
    float left = e * weight;
#pragma unroll
    for (int d = 0; d < 3; d++) {
      part[d][t] = __float_as_uint(left);
      left = left - __uint_as_float(part[d][t] & 0xffff0000u);
    }
  }
  asm volatile("" ::: "memory");
#pragma unroll
  for (int d = 0; d < 3; d++)
    *reinterpret_cast<uint2 *>(turn_to + 4 * d * kTurned) = make_uint2(upper(part[d][1], part[d][0]), upper(part[d][3], part[d][2]));
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  const v8bf low = *reinterpret_cast<const v8bf *>(turn_from), high = *reinterpret_cast<const v8bf *>(turn_from + 8);
  asm volatile("" ::: "memory");
#pragma unroll
  for (int d = 0; d < 4; d++) {
    u.acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(codes_of(s.v[d][0], s.v[d][1]), low, u.acc[d], 0, 0, 0);
    u.acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(codes_of(s.v[d][2], s.v[d][3]), high, u.acc[d], 0, 0, 0);
  }
}

// A wave's run of keys, 64 at a time. While one 64 keys are worked on, the next are on
// their way, and before them the pages of those after: no load is under a branch, so
// the waits count what is still out. stage[0] holds the first 64, `next` the pages of
// the second.
template <typename R, typename S, typename F, typename Step>
__device__ __forceinline__ void walk(R &reader, S (&stage)[2], F next, int begin, int end, const Step &step) {
  auto turn = [&](const S &now, S &then, int key0, auto more) {
    if constexpr (decltype(more)::value) {
      const F after = reader.find(key0 + 128);
      reader.load(next, key0 + 64, then);
      next = after;
    }
    step(now, key0);
  };
  const std::true_type more;
  const std::false_type no_more;
  int key0 = begin;
  for (; key0 + 128 < end; key0 += 128) {
    turn(stage[0], stage[1], key0, more);
    turn(stage[1], stage[0], key0 + 64, more);
  }
  if (key0 + 64 < end) {
    turn(stage[0], stage[1], key0, more);
    turn(stage[1], stage[0], key0 + 64, no_more);
  } else {
    turn(stage[0], stage[1], key0, no_more);
  }
}

//
// Over a shared prefix it is the keys from `base` on, in the parts behind the prefix's.
template <bool WIDE, typename Args>
__device__ __forceinline__ void attend(const Args &a, int block) {
  const Cache &c = a.c;
  int base = 0, own_parts = a.parts, first_part = 0;
  if constexpr (kShared<Args>) {
    base = a.base;
    own_parts = a.own_parts;
    first_part = a.first_part;
  }
  const bool whole = !kShared<Args> && own_parts == 1;  // no other part of a row: it is finished here
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Workgroups go to the 8 XCDs in turn: those of the key heads of one value head
  // follow one another on the same one, whose L2 then holds the values for all.
  const int share = c.key_heads / c.kv_heads, turn_of = block / 8;
  int task = (turn_of / share * 8 + block % 8) * share + turn_of % share;
  const int key_head = task % c.key_heads;
  task /= c.key_heads;
  const int tile = task % a.tiles;
  task /= a.tiles;
  const int part = task % own_parts, seq = task / own_parts;
  if (seq >= c.n_seqs) return;
  const int group = c.n_heads / c.key_heads;
  int len, first, n;
  bool bad;
  const int start = start_of(c, seq);
  if (!attend_span(a, seq, len, first, n, bad)) {
    if (bad && whole && tile == 0 && wave == 0) refuse_rows(a, seq, key_head * group, group);
    return;
  }
  const int limit = len + n, from_key = base + part * a.chunk;
  if (16 * tile >= group * n || from_key >= limit) return;
  // Waves: runs of the part's keys, in whole 64s, times quads of columns.
  const int columns = group * n, left = columns - 16 * tile;
  const int quads = left <= 4 ? 1 : left <= 8 ? 2 : 4, runs = 4 / quads, run = wave / quads, at_quad = wave % quads;
  const int to_key = from_key + a.chunk < limit ? from_key + a.chunk : limit;
  const int each = (to_key - from_key + 64 * runs - 1) / (64 * runs) * 64;
  const int begin = from_key + run * each, end = begin + each < to_key ? begin + each : to_key;
  const int column0 = 16 * tile + 4 * at_quad;

  Reader<WIDE> reader(c, seq, key_head, limit);
  Found next;
  Stage stage[2];
  Quad quad;
  quad.m = -__builtin_inff();
  quad.den = 0.0f;
#pragma unroll
  for (int d = 0; d < 4; d++) quad.acc[d] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  int power = -300;
  __shared__ __attribute__((aligned(16))) uint16_t turned[4][16 * kTurned];
  *reinterpret_cast<uint2 *>(turned[wave] + (12 + g) * kTurned + 4 * l16) = make_uint2(0, 0);
  const bool works = begin < end && column0 < columns;
  if (works) {
    next = reader.find(begin);
    // Column column0 + q: query row first + column % n, head key_head * group + column / n.
    float4 x[4];
    const int wanted = column0 + l16 / 4, column = wanted < columns ? wanted : columns - 1;
    const float *q = a.q + (static_cast<size_t>(first + column % n) * c.n_heads + key_head * group + column / n) * 64 + 16 * g;
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = reinterpret_cast<const float4 *>(q)[i];
    reader.load(next, begin, stage[0]);
    next = reader.find(begin + 64);
    quad.begin(x);
    const int mine = column0 + g;
    quad.visible = len + (mine < columns ? mine : columns - 1) % n + 1;
    walk(reader, stage, next, begin, end,
         [&](const Stage &now, int key0) { consume(quad, power, now, key0, reader.last_block, turned[wave]); });
  }
  if (__any(reader.missing) && lane == 0) c.refused[seq] = 1;
  // Asked here, where no load is waited for.
  if (overlaps(c, seq, first, start)) {
    if (whole && tile == 0 && wave == 0) refuse_rows(a, seq, key_head * group, group);
    return;
  }

  // The waves' states meet in LDS: [run][column], 16 in all.
  __shared__ float s_m[16], s_den[16];
  __shared__ __attribute__((aligned(16))) float s_o[16][68];
  quad.end(power, s_m + 4 * wave, s_den + 4 * wave, s_o + 4 * wave);
  __syncthreads();
  // Thread: a column and four dims.
  const int col = threadIdx.x / 16, dim = threadIdx.x % 16 * 4, wide = 4 * quads;
  const int out_column = 16 * tile + col;
  if (col >= wide || out_column >= columns) return;
  float top, total;
  const v4f o = join_runs(s_m, s_den, s_o, col, wide, runs, dim, top, total);
  const int out_head = key_head * group + out_column / n;
  const size_t out_row = static_cast<size_t>(first + out_column % n) * c.n_heads + out_head;
  if (whole) {
    const float factor = sink_factor(a.sinks, out_head, top, total);
    v4f y;
#pragma unroll
    for (int i = 0; i < 4; i++) y[i] = __fdiv_rn(o[i], total) * factor;
    *reinterpret_cast<v4f *>(a.out + out_row * 64 + dim) = y;
    return;
  }
  store_part(a, out_row * a.parts + first_part + part, dim, o, top, total);
}

template <bool WIDE>
__global__ __launch_bounds__(256, 3) void attend_kernel(AttendArgs a) {
  attend<WIDE>(a, blockIdx.x);
}

// What attend does for a part of a sequence and a key head, by one wave, four columns at a
// time: for many sequences of short lengths, as a launch over a shared prefix has room for two
// workgroups a compute unit, and one for each of 64 sequences and 16 key heads would wait.
template <bool WIDE>
__device__ __forceinline__ void attend_alone(const SharedArgs &a, int block) {
  const Cache &c = a.c;
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int task = 4 * block + wave;
  const int key_head = task % c.key_heads;
  task /= c.key_heads;
  const int part = task % a.own_parts, seq = task / a.own_parts;
  if (seq >= c.n_seqs) return;
  const int group = c.n_heads / c.key_heads;
  int len, first, n;
  bool bad;
  const int start = start_of(c, seq);
  if (!attend_span(a, seq, len, first, n, bad)) return;
  const int limit = len + n, columns = group * n, begin = a.base + part * a.chunk;
  const int end = begin + a.chunk < limit ? begin + a.chunk : limit;
  if (begin >= end) return;
  __shared__ __attribute__((aligned(16))) uint16_t turned[4][16 * kTurned];
  __shared__ float s_m[16], s_den[16];
  __shared__ __attribute__((aligned(16))) float s_o[16][68];
  *reinterpret_cast<uint2 *>(turned[wave] + (12 + g) * kTurned + 4 * l16) = make_uint2(0, 0);
  Reader<WIDE> reader(c, seq, key_head, limit);
  for (int column0 = 0; column0 < columns; column0 += 4) {
    Stage stage[2];
    Found next = reader.find(begin);
    float4 x[4];
    const int wanted = column0 + l16 / 4, column = wanted < columns ? wanted : columns - 1;
    const float *q = a.q + (static_cast<size_t>(first + column % n) * c.n_heads + key_head * group + column / n) * 64 + 16 * g;
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = reinterpret_cast<const float4 *>(q)[i];
    reader.load(next, begin, stage[0]);
    next = reader.find(begin + 64);
    Quad quad;
    int power = -300;
    quad.begin(x);
    const int mine = column0 + g;
    quad.visible = len + (mine < columns ? mine : columns - 1) % n + 1;
    walk(reader, stage, next, begin, end,
         [&](const Stage &now, int key0) { consume(quad, power, now, key0, reader.last_block, turned[wave]); });
    if (column0 == 0) {
      if (__any(reader.missing) && lane == 0) c.refused[seq] = 1;
      if (overlaps(c, seq, first, start)) return;
    }
    quad.end(power, s_m + 4 * wave, s_den + 4 * wave, s_o + 4 * wave);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    // Lane: a column and four dims.
    const int at = column0 + g, dim = 4 * l16;
    if (at < columns) {
      const size_t row = static_cast<size_t>(first + at % n) * c.n_heads + key_head * group + at / n;
      store_part(a, row * a.parts + a.first_part + part, dim, *reinterpret_cast<const v4f *>(&s_o[4 * wave + g][dim]), s_m[4 * wave + g],
                 s_den[4 * wave + g]);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
}

// ---- attention over a prefix that the batch shares ----------------------------------
// The rows of a call see positions below `base` in the pages of one sequence, the
// prefix, each row all of them, so all rows' queries of a key head are columns of the same
// products, and the keys are read once for 32 columns. What a row sees behind `base` are its
// own sequence's positions (attend), and merge_kernel joins both: with states (m_i, d_i, o_i)
// of disjoint keys, m = max m_i, o = sum 2^(m_i - m) o_i / sum 2^(m_i - m) d_i.
//
// A wave takes 32 columns and 64 keys at a time, on the matrix instructions of 32 by 32.
// Scores. Lane (l32, h) has column l32's query as two FP16 numbers an element, scaled so that the
// largest is in [2^13, 2^14). The rest after the first has up to 12 bits and a sign where FP16
// has 11, so an element is off by up to 2^-23 of itself, or half an FP16 subnormal step, 2^-38 of the
// largest. Codes are FP16 numbers, so products are exact and their sums round as FP32's. Row m of
// key tile t is position m % 4 + 4 (m / 8) of block 2 t + m / 4 % 2, so that lane (l32, h)
// gets the scores of column l32 with the 16 keys of blocks h and 2 + h, a scale for each.
// Weights. exp2(s - m) times the block's value scale is three BF16 numbers, as in consume, which
// stand where the second product takes them; its other operand is the value codes of dim
// l32 (and 32 + l32) as they stand, as BF16 numbers.
//
// Bound: the vector instructions, 605 for 64 keys, of which the codes' conversion is 176
// and the weights' exponentials and parts 300, and the matrix instructions' 1,280 cycles, which
// hide behind them in part only. 200 rows over 32,768 positions (8 key heads, 105 million
// scores) and then each sequence's own take 111 us with the merge; the matrix products alone
// are 27. The same with 16 columns a wave takes 5 % longer; with scores of one step more in
// flight, weights' parts by sums of two products, or the scheduler told to mix both kinds it is
// no faster. Reading each sequence's copy of the prefix would be 33 MB a sequence.
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));

// Eight codes as FP16 numbers: 1024 + 128 + code has the code, its top bit turned, in its
// low byte.
__device__ __forceinline__ v8h halves_of(int first, int second) {
  const uint32_t w[2] = {static_cast<uint32_t>(first) ^ 0x80808080u, static_cast<uint32_t>(second) ^ 0x80808080u};
  v4i to;
#pragma unroll
  for (int i = 0; i < 2; i++)
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const uint32_t bits = __builtin_amdgcn_perm(0x64646464u, w[i], j == 0 ? 0x04010400u : 0x04030402u);
      to[2 * i + j] = __builtin_bit_cast(int, __builtin_bit_cast(v2h, bits) - v2h{static_cast<_Float16>(1152.0f), static_cast<_Float16>(1152.0f)});
    }
  return __builtin_bit_cast(v8h, to);
}

// The sequence of each of a tile's rows row0 .. row0 + rows - 1 that one which takes part
// has, by the threads of a workgroup or wave; `owner` begins at -1. False if none was found.
// Of several it is the first: where one of them is accepted, those behind it overlap it and
// are refused, and one before it would have had it refused.
__device__ __forceinline__ bool find_owners(const SharedArgs &a, int row0, int rows, int *owner, int thread, int threads) {
  const Cache &c = a.c;
  const int seq0 = c.row_start ? 0 : row0, seq_end = c.row_start ? c.n_seqs : row0 + rows;
  bool any = false;
  for (int seq = seq0 + thread; seq < seq_end; seq += threads) {
    int len, first, n;
    bool bad;
    if (!attend_span(a, seq, len, first, n, bad)) continue;
    for (int r = first > row0 ? first : row0; r < first + n && r < row0 + rows; r++) {
      atomicMin(reinterpret_cast<uint32_t *>(owner + (r - row0)), static_cast<uint32_t>(seq));  // -1 is the largest
      any = true;
    }
  }
  return any;
}

struct Stage32 {
  v4i k[2][2], v[2][2];  // [key tile][16 dims 2 j + h], [key tile][32 dims]
  float k_scale[2], v_scale[2];  // of block 2 t + h
};
template <bool WIDE>
struct Reader32 {
  struct Pages {
    int k[2], v[2];
  };
  const Cache &c;
  const int32_t *table;
  int key_head, value_head, last_block;
  bool missing = false;

  __device__ __forceinline__ Reader32(const Cache &cache, int seq, int head, int limit)
      : c(cache), table(cache.table + static_cast<size_t>(seq) * cache.seq_pages), key_head(head),
        value_head(head * cache.kv_heads / cache.key_heads), last_block((limit - 1) / kBlock) {}

  __device__ __forceinline__ int held(int block) const { return block < last_block ? block : last_block; }
  __device__ __forceinline__ Pages find(int key0) const {
    typedef __attribute__((address_space(4))) const int32_t scalar_table;  // read by scalar loads
    const int b = key0 / kBlock;
    Pages f;
    if constexpr (WIDE) {
      f.k[0] = f.k[1] = f.v[0] = f.v[1] = reinterpret_cast<scalar_table *>(reinterpret_cast<uintptr_t>(table))[held(b) >> c.shift];
    } else {
      const int of_k = threadIdx.x >> 2 & 1, of_v = threadIdx.x >> 5 & 1;
#pragma unroll
      for (int t = 0; t < 2; t++) {
        f.k[t] = table[held(b + 2 * t + of_k) >> c.shift];
        f.v[t] = table[held(b + 2 * t + of_v) >> c.shift];
      }
    }
    return f;
  }
  __device__ __forceinline__ void load(const Pages &f, int key0, Stage32 &s) {
    const int l32 = threadIdx.x & 31, h = threadIdx.x >> 5 & 1, of_k = l32 >> 2 & 1, mask = (1 << c.shift) - 1;
    const int b = key0 / kBlock;
    const int k_lane = (l32 & 3) * 256 + (l32 >> 3) * 64 + 16 * h, v_lane = l32 * 16;
#pragma unroll
    for (int t = 0; t < 2; t++) {
      missing |= f.k[t] < 0;
      const long kp = f.k[t] < 0 ? 0 : f.k[t], vp = f.v[t] < 0 ? 0 : f.v[t];
      const int8_t *k, *v;
      if constexpr (WIDE) {
        const long kn = ((kp * c.key_heads + key_head) << c.shift) + (b & mask) + 2 * t;
        const long vn = ((vp * c.kv_heads + value_head) << c.shift) + (b & mask) + 2 * t;
        k = c.k_codes + kn * kBlockBytes + (of_k * kBlockBytes + k_lane);
        v = c.v_codes + vn * kBlockBytes + (h * kBlockBytes + v_lane);
        s.k_scale[t] = (c.k_scales + kn)[h];
        s.v_scale[t] = (c.v_scales + vn)[h];
      } else {
        const int v_in = held(b + 2 * t + h) & mask;
        const long vn = ((vp * c.kv_heads + value_head) << c.shift) + v_in;
        k = c.k_codes + (((kp * c.key_heads + key_head) << c.shift) + (held(b + 2 * t + of_k) & mask)) * kBlockBytes + k_lane;
        v = c.v_codes + vn * kBlockBytes + v_lane;
        s.k_scale[t] = c.k_scales[((vp * c.key_heads + key_head) << c.shift) + v_in];
        s.v_scale[t] = c.v_scales[vn];
      }
      s.k_scale[t] = f.v[t] < 0 ? __builtin_nanf("") : s.k_scale[t];
#pragma unroll
      for (int j = 0; j < 2; j++) {
        s.k[t][j] = *reinterpret_cast<const v4i *>(k + 32 * j);
        s.v[t][j] = *reinterpret_cast<const v4i *>(v + 512 * j);
      }
    }
  }
};

typedef float v16f __attribute__((ext_vector_type(16)));

__device__ __forceinline__ float halves_max(float v) {
  const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __builtin_fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
}

struct Columns32 {
  v8h q[2][4];  // the two parts of dims 16 (2 j + h) + 8 i .. + 7, at 2 j + i
  float factor, m, den;
  v16f acc[2];  // dims 32 d + 8 (i / 4) + 4 h + i % 4
  int power;

  __device__ __forceinline__ void clear() {
    m = -__builtin_inff();
    den = 0.0f;
    power = -300;
#pragma unroll
    for (int d = 0; d < 2; d++)
#pragma unroll
      for (int i = 0; i < 16; i++) acc[d][i] = 0.0f;
  }
  // From dims 16 (2 j + h) .. + 15 of the lane's column.
  __device__ __forceinline__ void begin(const float4 (&x)[2][4]) {
    uint32_t big = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const float y[4] = {x[i / 4][i % 4].x, x[i / 4][i % 4].y, x[i / 4][i % 4].z, x[i / 4][i % 4].w};
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const uint32_t bits = __float_as_uint(y[j]) & 0x7fffffffu;
        big = bits > big ? bits : big;
      }
    }
    const auto p = __builtin_amdgcn_permlane32_swap(big, big, false, false);
    big = p[0] > p[1] ? p[0] : p[1];
    const bool finite = big < 0x7f800000u;
    int e = !finite || big == 0 ? 0 : __builtin_amdgcn_frexp_expf(__uint_as_float(big));
    e = e < -90 ? -90 : e;
    // log2(e) / 8: scores in powers of two.
    factor = finite ? __builtin_ldexpf(0.180336880111120426f, e - 14) : __builtin_nanf("");
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const float y[4] = {x[i / 4][i % 4].x, x[i / 4][i % 4].y, x[i / 4][i % 4].z, x[i / 4][i % 4].w};
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float scaled = finite ? __builtin_ldexpf(y[j], 14 - e) : 0.0f;
        const _Float16 high = static_cast<_Float16>(scaled);
        q[0][i / 2][i % 2 * 4 + j] = high;
        q[1][i / 2][i % 2 * 4 + j] = static_cast<_Float16>(scaled - static_cast<float>(high));
      }
    }
  }

  __device__ __forceinline__ void consume(const Stage32 &s, int key0, int last_block) {
    const int h = threadIdx.x >> 5 & 1;
    const float ninf = -__builtin_inff();
    bool none[2];
    float k_scale[2], v_scale[2];
#pragma unroll
    for (int t = 0; t < 2; t++) {
      none[t] = key0 / kBlock + 2 * t + h > last_block;  // a block behind the last
      const float v = none[t] ? 0.0f : s.v_scale[t];
      k_scale[t] = v != v ? __builtin_nanf("") : s.k_scale[t];
      v_scale[t] = v != v ? 0.0f : v;
    }
    const float widest = halves_max(__builtin_fmaxf(v_scale[0], v_scale[1]));
    int above = widest > 0.0f ? __builtin_amdgcn_frexp_expf(widest) : -300;
    above = __builtin_amdgcn_readfirstlane(above > power ? above : power);
    const int lower = power - above;
    power = above;
    v16f sums[2];
#pragma unroll
    for (int t = 0; t < 2; t++) {
      v16f sum;
#pragma unroll
      for (int i = 0; i < 16; i++) sum[i] = 0.0f;
#pragma unroll
      for (int j = 0; j < 2; j++) {
        const v8h first = halves_of(s.k[t][j][0], s.k[t][j][1]), second = halves_of(s.k[t][j][2], s.k[t][j][3]);
#pragma unroll
        for (int part = 1; part >= 0; part--) {
          sum = __builtin_amdgcn_mfma_f32_32x32x16_f16(first, q[part][2 * j], sum, 0, 0, 0);
          sum = __builtin_amdgcn_mfma_f32_32x32x16_f16(second, q[part][2 * j + 1], sum, 0, 0, 0);
        }
      }
      sums[t] = sum;
    }
    float scale[2], top = ninf;
#pragma unroll
    for (int t = 0; t < 2; t++) {
      scale[t] = none[t] ? 0.0f : factor * k_scale[t];
      float most = sums[t][0];
#pragma unroll
      for (int i = 1; i < 16; i++) most = __builtin_fmaxf(most, sums[t][i]);
      top = __builtin_fmaxf(top, none[t] ? ninf : most * scale[t]);
    }
    top = __builtin_fmaxf(m, halves_max(top));
    const float from = top == ninf ? 0.0f : top;
    if (__any(top > m) || lower < 0) {
      const float keep = __builtin_amdgcn_exp2f(m - from), scaled = __builtin_ldexpf(keep, lower);
      den = den * keep;
#pragma unroll
      for (int d = 0; d < 2; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) acc[d][i] = acc[d][i] * scaled;
      m = top;
    }
#pragma unroll
    for (int t = 0; t < 2; t++) {
      const float minus = none[t] ? ninf : -from, weight = __builtin_ldexpf(v_scale[t], 64 - power);
#pragma unroll
      for (int half = 0; half < 2; half++) {
        // Positions 8 half .. + 7 of block 2 t + h.
        v4i words[3];
#pragma unroll
        for (int pair = 0; pair < 4; pair++) {
          uint32_t bits[3][2];
#pragma unroll
          for (int j = 0; j < 2; j++) {
            const float e = __builtin_amdgcn_exp2f(fmaf_(sums[t][8 * half + 2 * pair + j], scale[t], minus));
            den = den + e;
            float left = e * weight;
#pragma unroll
            for (int d = 0; d < 3; d++) {
              bits[d][j] = __float_as_uint(left);
              left = left - __uint_as_float(bits[d][j] & 0xffff0000u);
            }
          }
#pragma unroll
          for (int d = 0; d < 3; d++) words[d][pair] = static_cast<int>(upper(bits[d][1], bits[d][0]));
        }
        v8bf codes[2];
#pragma unroll
        for (int d = 0; d < 2; d++) codes[d] = codes_of(s.v[t][d][2 * half], s.v[t][d][2 * half + 1]);
#pragma unroll
        for (int part = 2; part >= 0; part--)
#pragma unroll
          for (int d = 0; d < 2; d++)
            acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(codes[d], __builtin_bit_cast(v8bf, words[part]), acc[d], 0, 0, 0);
      }
    }
  }
};

// What a wave of the prefix's kernels has: its columns from column0 on, of rows from row0 on
// with these owners, and keys begin .. end - 1. `at`: the lane's column's number among
// all rows and heads.
template <bool WIDE>
__device__ __forceinline__ void walk_prefix(const SharedArgs &a, Columns32 &state, int key_head, bool live, size_t at, int rows,
                                            const int *owner, int begin, int end) {
  const Cache &c = a.c;
  const int lane = threadIdx.x & 63, h = lane >> 5;
  Reader32<WIDE> reader(c, a.prefix, key_head, a.base);
  Stage32 stage[2];
  auto next = reader.find(begin);
  float4 x[2][4];
#pragma unroll
  for (int j = 0; j < 2; j++)
#pragma unroll
    for (int i = 0; i < 4; i++)
      x[j][i] = live ? reinterpret_cast<const float4 *>(a.q + at * 64 + 16 * (2 * j + h))[i] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  reader.load(next, begin, stage[0]);
  next = reader.find(begin + 64);
  state.begin(x);
  walk(reader, stage, next, begin, end, [&](const Stage32 &now, int key0) { state.consume(now, key0, reader.last_block); });
  if (__any(reader.missing))
    for (int r = lane; r < rows; r += 64)
      if (owner[r] >= 0) c.refused[owner[r]] = 1;
  const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(state.den), __float_as_uint(state.den), false, false);
  state.den = __uint_as_float(both[0]) + __uint_as_float(both[1]);
}

// Up to 64 columns: a workgroup for a part of the keys, its four waves side by side over
// the columns (`beside` of them) and the part's runs.
template <bool WIDE>
__device__ __forceinline__ void attend_prefix_few(const SharedArgs &a) {
  const Cache &c = a.c;
  const int lane = threadIdx.x & 63, l32 = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // The key heads of one value head follow one another on one XCD.
  const int share = c.key_heads / c.kv_heads, turn_of = blockIdx.x / 8;
  const int task = turn_of / share * 8 + blockIdx.x % 8;
  const int key_head = task % c.kv_heads * share + turn_of % share, part = task / c.kv_heads;
  if (part >= a.first_part) return;
  const int group = c.n_heads / c.key_heads, columns = group * c.rows;
  const int beside = a.beside, across = 32 * beside, runs = 4 / beside, run = wave / beside;
  __shared__ int owner[64];
  if (threadIdx.x < 64) owner[threadIdx.x] = -1;
  __syncthreads();
  if (!__syncthreads_or(find_owners(a, 0, c.rows, owner, threadIdx.x, 256))) return;
  const int from_key = part * a.prefix_chunk, to_key = from_key + a.prefix_chunk < a.base ? from_key + a.prefix_chunk : a.base;
  const int each = (to_key - from_key + 64 * runs - 1) / (64 * runs) * 64;
  const int begin = from_key + run * each, end = begin + each < to_key ? begin + each : to_key;
  const int column = wave % beside * 32 + l32, row = column / group;
  const bool live = column < columns && owner[row] >= 0;
  Columns32 state;
  state.clear();
  if (begin < end && __any(live))
    walk_prefix<WIDE>(a, state, key_head, live, static_cast<size_t>(row) * c.n_heads + key_head * group + column % group, c.rows,
                      owner, begin, end);
  // The waves' states meet in LDS: [run][column].
  __shared__ float s_m[128], s_den[128];
  __shared__ __attribute__((aligned(16))) float s_o[128][68];
  const int to = 32 * wave + l32;
  if (h == 0) {
    s_m[to] = state.m;
    s_den[to] = state.den;
  }
#pragma unroll
  for (int d = 0; d < 2; d++)
#pragma unroll
    for (int i = 0; i < 4; i++) {
      v4f o;
#pragma unroll
      for (int j = 0; j < 4; j++) o[j] = __builtin_ldexpf(state.acc[d][4 * i + j], state.power - 64);
      *reinterpret_cast<v4f *>(&s_o[to][32 * d + 8 * i + 4 * h]) = o;
    }
  __syncthreads();
  const int dim = threadIdx.x % 16 * 4;
  for (int at = threadIdx.x / 16; at < columns; at += 16) {
    if (owner[at / group] < 0) continue;
    float top, total;
    const v4f o = join_runs(s_m, s_den, s_o, at, across, runs, dim, top, total);
    const size_t slot = (static_cast<size_t>(at / group) * c.n_heads + key_head * group + at % group) * a.parts + part;
    store_part(a, slot, dim, o, top, total);
  }
}

// More columns: every wave has 32 of them and a part of the keys to itself, so that any
// number of columns leaves no wave idle. Waves follow one another by column, key head of
// one value head, then part and value head, and each XCD has a stretch of them.
template <bool WIDE>
__device__ __forceinline__ void attend_prefix(const SharedArgs &a) {
  const Cache &c = a.c;
  const int lane = threadIdx.x & 63, l32 = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int share = c.key_heads / c.kv_heads, group = c.n_heads / c.key_heads, columns = group * c.rows;
  int task = (blockIdx.x % 8 * (a.prefix_blocks / 8) + blockIdx.x / 8) * 4 + wave;
  const int tile = task % a.prefix_tiles;
  task /= a.prefix_tiles;
  const int sharer = task % share;
  task /= share;
  const int key_head = task % c.kv_heads * share + sharer, part = task / c.kv_heads;
  if (part >= a.first_part) return;
  const int column0 = 32 * tile, row0 = column0 / group, row_end = (column0 + 31) / group + 1;
  const int rows = (row_end < c.rows ? row_end : c.rows) - row0;
  __shared__ int all_owners[4][32];
  int *const owner = all_owners[wave];
  if (lane < 32) owner[lane] = -1;
  asm volatile("" ::: "memory");
  if (!__any(find_owners(a, row0, rows, owner, lane, 64))) return;
  asm volatile("" ::: "memory");
  const int begin = part * a.prefix_chunk, end = begin + a.prefix_chunk < a.base ? begin + a.prefix_chunk : a.base;
  // The lane's column: row column / group, head key_head * group + column % group. One that
  // is no row's has a query of zeros, and is left out in the end.
  const int column = column0 + l32, row = column / group;
  const bool live = column < columns && owner[row - row0] >= 0;
  const size_t at = static_cast<size_t>(row) * c.n_heads + key_head * group + column % group;
  Columns32 state;
  state.clear();
  walk_prefix<WIDE>(a, state, key_head, live, at, rows, owner, begin, end);
  if (!live) return;
  const size_t slot = at * a.parts + part;
#pragma unroll
  for (int d = 0; d < 2; d++)
#pragma unroll
    for (int i = 0; i < 4; i++) {
      v4f o;
#pragma unroll
      for (int j = 0; j < 4; j++) o[j] = __builtin_ldexpf(state.acc[d][4 * i + j], state.power - 64);
      store_part(a, slot, 32 * d + 8 * i + 4 * h, o, state.m, state.den);
    }
}

// Both in one launch, the prefix's workgroups first: they take longer, and where their
// vector instructions are the bound, the sequences' own keys come from memory meanwhile.
template <bool WIDE, bool FEW>
__global__ __launch_bounds__(256, 2) void shared_kernel(SharedArgs a) {
  const int block = static_cast<int>(blockIdx.x) - a.prefix_blocks;
  if (block >= 0 && a.alone)
    attend_alone<WIDE>(a, block);
  else if (block >= 0)
    attend<WIDE>(a, block);
  else if constexpr (FEW)
    attend_prefix_few<WIDE>(a);
  else
    attend_prefix<WIDE>(a);
}

// The parts of a sequence's rows of one head: as many of the waves for each row as
// there are, lane = element, eight parts of a wave in flight. Bound by the launch and
// the trips to memory: 4.4 us for 7 parts of 25 rows, 5.3 for 57 parts of two.
template <int WAVES, typename Args>
__global__ __launch_bounds__(64 * WAVES) void merge_kernel(Args a) {
  const Cache &c = a.c;
  constexpr int BATCH = 8;
  const int head = blockIdx.x, seq = blockIdx.y;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  __shared__ float s_m[WAVES], s_den[WAVES], s_o[WAVES][64];
  int len, first, n;
  bool bad;
  const int start = start_of(c, seq);
  const bool live = attend_span(a, seq, len, first, n, bad);
  if (bad && wave == 0) refuse_rows(a, seq, head, 1);
  if (!live) return;
  const int spread = n == 1 ? 1 : n == 2 ? 2 : n <= 4 ? 4 : 8;
  const int waves = spread < WAVES ? WAVES / spread : 1, own = wave % waves;
  int parts = (len + n - 1) / a.chunk + 1;
  if constexpr (kShared<Args>) parts = a.first_part + (len + n - a.base - 1) / a.chunk + 1;
  for (int r0 = 0; r0 < n; r0 += WAVES / waves) {
    const int r = r0 + wave / waves;
    const size_t row = static_cast<size_t>(first + (r < n ? r : 0)) * c.n_heads + head, at = row * a.parts;
    const float2 *md = reinterpret_cast<const float2 *>(a.part_md) + at;
    const float *part_o = a.part_o + at * 64 + lane;
    float m = -__builtin_inff(), den = 0.0f, o = 0.0f;
    if (r < n)
      for (int p = own; p < parts; p += waves * BATCH) {
        float2 v[BATCH];
        float x[BATCH];
#pragma unroll
        for (int i = 0; i < BATCH; i++) {
          const int q = p + waves * i;
          v[i] = md[q < parts ? q : p];
          x[i] = part_o[static_cast<size_t>(q < parts ? q : p) * 64];
        }
        float top = m;
#pragma unroll
        for (int i = 0; i < BATCH; i++) top = __builtin_fmaxf(top, v[i].x);
        const float keep = state_weight(m, den, top);
        den = den * keep;
        o = o * keep;
#pragma unroll
        for (int i = 0; i < BATCH; i++)
          if (p + waves * i < parts) {
            const float f = state_weight(v[i].x, v[i].y, top);
            den = fmaf_(v[i].y, f, den);
            o = fmaf_(x[i], f, o);
          }
        m = top;
      }
    if (lane == 0) {
      s_m[wave] = m;
      s_den[wave] = den;
    }
    s_o[wave][lane] = o;
    __syncthreads();
    if (own == 0 && r < n && !overlaps(c, seq, first, start)) {
      float top = m;
      for (int w = 1; w < waves; w++) top = __builtin_fmaxf(top, s_m[wave + w]);
      float total = 0.0f;
      o = 0.0f;
      for (int w = 0; w < waves; w++) {
        const float f = state_weight(s_m[wave + w], s_den[wave + w], top);
        total = fmaf_(s_den[wave + w], f, total);
        o = fmaf_(s_o[wave + w][lane], f, o);
      }
      a.out[row * 64 + lane] = __fdiv_rn(o, total) * sink_factor(a.sinks, head, top, total);
    }
    __syncthreads();
  }
  if (wave == 0 && overlaps(c, seq, first, start)) refuse_rows(a, seq, head, 1);
}

// ---- pages of a sequence ---------------------------------------------------------
constexpr int kMapped = 240;
struct MapArgs {
  int32_t *table, *tags;  // of the sequence
  int first, count, shift, heads;
  int32_t pages[kMapped];
};

// Writes table entries, and forgets the FP32 blocks that stood where other pages come.
__global__ __launch_bounds__(256) void map_kernel(MapArgs a) {
  for (int i = threadIdx.x; i < 2 * a.heads; i += 256) {
    const int block = a.tags[i], at = block >> a.shift;
    if (block >= 0 && at >= a.first && at < a.first + a.count && a.table[at] != a.pages[at - a.first]) a.tags[i] = -1;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < a.count; i += 256) a.table[a.first + i] = a.pages[i];
}

__global__ __launch_bounds__(256) void fill_kernel(int32_t *to, size_t count, int32_t value) {
  for (size_t i = blockIdx.x * static_cast<size_t>(256) + threadIdx.x; i < count; i += static_cast<size_t>(gridDim.x) * 256)
    to[i] = value;
}

void free_pages(Pages *kv) {
  void *buffers[] = {kv->k_codes,   kv->v_codes, kv->k_scales, kv->v_scales, kv->k_writers,
                     kv->v_writers, kv->table,   kv->open,     kv->tags,     kv->refused};
  for (void *p : buffers)
    if (p) (void)hipFree(p);
}

Cache cache_of(const Pages *kv, size_t rows, const int32_t *row_start, const int32_t *lens, size_t n_seqs) {
  Cache c = {};
  c.k_codes = kv->k_codes;
  c.v_codes = kv->v_codes;
  c.k_scales = kv->k_scales;
  c.v_scales = kv->v_scales;
  c.k_writers = kv->k_writers;
  c.v_writers = kv->v_writers;
  c.table = kv->table;
  c.open = kv->open;
  c.tags = kv->tags;
  c.refused = kv->refused;
  c.shift = kv->shift;
  c.seq_pages = static_cast<int>(kv->seq_pages);
  c.n_heads = static_cast<int>(kv->n_heads);
  c.key_heads = static_cast<int>(kv->key_heads);
  c.kv_heads = static_cast<int>(kv->kv_heads);
  c.row_start = row_start;
  c.lens = lens;
  c.rows = static_cast<int>(rows);
  c.n_seqs = static_cast<int>(n_seqs);
  return c;
}

// What every call over a batch checks.
int check_batch(const char *name, const Ctx *ctx, const Pages *kv, size_t rows, const int32_t *row_start,
                const int32_t *lens, size_t n_seqs) {
  FOCR_REQUIRE(ctx && kv, FOCR_E_ARG, std::string(name) + ": null argument");
  FOCR_REQUIRE(kv->device == ctx->device, FOCR_E_ARG, std::string(name) + ": the cache is on another device than the context");
  FOCR_REQUIRE(n_seqs <= kv->n_seqs, FOCR_E_SHAPE, std::string(name) + ": more sequences than the cache has");
  FOCR_REQUIRE(rows < (size_t(1) << 24), FOCR_E_SHAPE, std::string(name) + ": too many rows");
  FOCR_REQUIRE(row_start || rows == n_seqs, FOCR_E_SHAPE, std::string(name) + ": without row_start every sequence has one row");
  FOCR_REQUIRE(rows == 0 || n_seqs == 0 || lens, FOCR_E_ARG, std::string(name) + ": null lengths");
  return FOCR_OK;
}

int launch_append(Ctx *ctx, AppendArgs a, bool qkv) {
  const Cache &c = a.c;
  // Units: n rows touch at most (n + 14) / 16 + 1 blocks, three of which are one
  // unit, so at most n / 16 units, or one.
  const int units = c.row_start ? c.rows / kBlock + (c.rows < c.n_seqs ? c.rows : c.n_seqs) : c.n_seqs;
  const int heads = a.positions ? c.n_heads + c.kv_heads : c.key_heads + c.kv_heads + (qkv ? c.n_heads : 0);
  FOCR_HIP_CHECK(hipSetDevice(ctx->device));
  const unsigned groups = static_cast<unsigned>((heads + 3) / 4);
  // Long prompts are near (us a call with its reading back, near / not: four of up to
  // 6,544 rows 89 / 104, one of 1,500 17.5 / 18.7; sixteen of up to 300 23.7 / 22.8, 200
  // of up to five 26.4 / 25.5: a sequence's first unit has three blocks' work), by the
  // mean over all the call's sequences: one prompt among many idle ones is not.
  a.near = c.rows / c.n_seqs >= 1024;
  dim3 grid(static_cast<unsigned>(units), groups);
  if (a.near) {
    const unsigned eights = static_cast<unsigned>((units + 7) / 8), y = std::min(eights, 32768u);
    grid = dim3(8 * groups, y, (eights + y - 1) / y);
  }
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, ctx->stream, a); };
  if (a.positions)
    launch(a.axes == 1 ? turn_kernel<1> : a.axes == 2 ? turn_kernel<2> : a.axes == 3 ? turn_kernel<3> : turn_kernel<4>);
  else
    launch(qkv ? append_kernel<true> : append_kernel<false>);
  FOCR_HIP_CHECK(hipGetLastError());
  return FOCR_OK;
}

// Attention, where shared > 0 over that many positions of sequence `prefix` first.
int launch_attend(const char *name, Ctx *ctx, const Pages *kv, const float *q, size_t rows, const int32_t *row_start,
                  const int32_t *lens, size_t n_seqs, size_t max_len, size_t prefix, size_t shared, const float *sinks,
                  float *out) {
  int rc = check_batch(name, ctx, kv, rows, row_start, lens, n_seqs);
  if (rc != FOCR_OK) return rc;
  FOCR_REQUIRE(prefix < kv->n_seqs, FOCR_E_SHAPE, std::string(name) + ": the cache has no such sequence");
  FOCR_REQUIRE(shared % kv->page == 0 && shared <= kv->seq_pages * kv->page, FOCR_E_SHAPE,
               std::string(name) + ": the shared positions are whole pages of a sequence");
  if (rows == 0 || n_seqs == 0) return FOCR_OK;
  FOCR_REQUIRE(q && out, FOCR_E_ARG, std::string(name) + ": null buffer");
  FOCR_REQUIRE(max_len > shared && max_len <= kv->seq_pages * kv->page, FOCR_E_SHAPE,
               std::string(name) + ": max_len is more than the shared positions, up to what a sequence's pages hold");
  SharedArgs a = {};
  a.c = cache_of(kv, rows, row_start, lens, n_seqs);
  a.q = q;
  a.sinks = sinks;
  a.out = out;
  a.max_len = static_cast<int>(max_len);
  a.base = static_cast<int>(shared);
  a.prefix = static_cast<int>(prefix);
  const size_t most = row_start ? std::min<size_t>(rows, 8) : 1;
  const size_t group = kv->n_heads / kv->key_heads, own = max_len - shared;
  a.tiles = static_cast<int>((group * most + 15) / 16);
  // Parts of whole 256 keys, at most 4,096 up to a million positions. Few sequences
  // need only fill the chip (us a call with 512 / 1,024 / 2,048 workgroups: one of
  // 131,072 positions 32.9 / 36.8 / 37.7, four of up to 16,000 16.3 / 17.8 / 18.8; six of
  // up to 3,000 with up to 8 rows 17.6 / 15.4 / 15.9); more, of different lengths, want
  // parts to spare (20 of up to 9,000 49.0 / 47.1 / 44.7, 40 of up to 5,000 with up to 8
  // rows 84.7 / 84.8 / 63.7).
  // Beside a prefix, many sequences of few columns and short lengths of their own have a wave a
  // part (us a call with a workgroup / a wave: 64 of one row and up to 300 positions 25.5 / 21.8,
  // 200 50.5 / 39.3, 32 19.7 / 14.6; of up to 1,000 64 26.5 / 24.5, of up to 4,000 48.9 / 55.7;
  // with eight columns and 1,000 36.1 / 44.9; 16 sequences as they were), 1,024 waves (2,048:
  // 25.6 for the first, 38.4, 14.4).
  const size_t units = n_seqs * kv->key_heads;
  a.alone = shared > 0 && units > 256 && rows * group <= 4 * n_seqs && own <= 1024;
  const size_t tasks = a.alone ? units : units * a.tiles;
  const size_t enough = n_seqs <= 2 ? 512 : n_seqs <= 8 || shared > 0 ? 1024 : 2048;
  const size_t want = tasks >= enough ? 1 : enough / tasks;
  const size_t chunk = std::max(std::min<size_t>((own + want - 1) / want, 4096), (own + kMaxParts - 1) / kMaxParts);
  a.chunk = static_cast<int>((chunk + 255) / 256 * 256);
  a.own_parts = static_cast<int>((own + a.chunk - 1) / a.chunk);
  const size_t share = kv->key_heads / kv->kv_heads;
  const size_t grid = a.alone ? (tasks * a.own_parts + 3) / 4 : (tasks * a.own_parts + 8 * share - 1) / (8 * share) * (8 * share);
  FOCR_REQUIRE(grid < (size_t(1) << 31), FOCR_E_SHAPE, std::string(name) + ": too many sequences and heads");
  bool few = false;
  if (shared > 0) {
    const size_t columns = group * rows;
    few = columns <= 64;
    // A workgroup, or a wave, for each compute unit or SIMD: the vector instructions are the
    // bound, and one wave has them busy (us a call with 128 / 256 / 512 workgroups: 8
    // sequences with up to 5 rows over 6,528 17.0 / 14.8 / 18.0, 64 with one 23.7 / 24.7 / 26.6, 4
    // over 30,016 32.0 / 22.4 / 23.7; with 1,024 / 2,048 / 4,096 waves: 200 over 32,768
    // 105 / 110 / 118, 100 with two rows over 8,192 41.8 / 44.8 / 52.2).
    a.beside = columns <= 32 ? 1 : 2;
    const size_t tiles = few ? 1 : (columns + 31) / 32, all = few ? 256 : 1024;
    const size_t each = kv->key_heads * tiles, parts = each >= all ? 1 : all / each;
    // At most 4,096 keys a part up to a million, as their sums' roundings add up (3,648 keys: 6e-7
    // of the result, 256: 2e-7).
    const size_t prefix_chunk = std::max(std::min<size_t>((shared + parts - 1) / parts, 4096), (shared + kMaxParts - 1) / kMaxParts);
    a.prefix_chunk = static_cast<int>((prefix_chunk + 63) / 64 * 64);
    a.first_part = static_cast<int>((shared + a.prefix_chunk - 1) / a.prefix_chunk);
    a.prefix_tiles = static_cast<int>(tiles);
    const size_t blocks = few ? (kv->kv_heads * a.first_part + 7) / 8 * 8 * share : (each * a.first_part + 31) / 32 * 8;
    FOCR_REQUIRE(blocks + grid < (size_t(1) << 31), FOCR_E_SHAPE, std::string(name) + ": too many rows and heads");
    a.prefix_blocks = static_cast<int>(blocks);
  }
  a.parts = a.first_part + a.own_parts;
  const size_t slots = rows * kv->n_heads * a.parts;
  FOCR_HIP_CHECK(hipSetDevice(ctx->device));
  if (a.parts > 1) {
    rc = ensure_scratch(ctx, slots * 66 * sizeof(float));
    if (rc != FOCR_OK) return rc;
    a.part_o = static_cast<float *>(ctx->scratch);
    a.part_md = a.part_o + slots * 64;
  }
  const bool wide = kv->page >= 64;
  const AttendArgs &alone = a;
  auto launch = [&](auto kernel, const auto &args) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(a.prefix_blocks + grid)), dim3(256), 0, ctx->stream, args);
  };
  if (shared == 0)
    launch(wide ? attend_kernel<true> : attend_kernel<false>, alone);
  else if (few)
    launch(wide ? shared_kernel<true, true> : shared_kernel<false, true>, a);
  else
    launch(wide ? shared_kernel<true, false> : shared_kernel<false, false>, a);
  FOCR_HIP_CHECK(hipGetLastError());
  if (a.parts > 1) {
    const dim3 each(static_cast<unsigned>(kv->n_heads), static_cast<unsigned>(n_seqs));
    // Parts of all a sequence's rows (us a call with 4 / 16 waves: 26 parts of one row
    // 9.8 / 10.4, 3 of one in 64 sequences 112 / 120; 57 of two 34.8 / 32.8, 59 of
    // eight 33.3 / 20.3).
    // Over a shared prefix by a sequence's mean rows, and 16 only for few sequences (17 parts of
    // up to five rows in 8: 18.6 / 14.8; of one in 64 24.7 / 35.8; ten of five in 32 24.7 / 26.1).
    const size_t mean = (rows + n_seqs - 1) / n_seqs;
    const bool four = shared > 0 ? n_seqs * kv->n_heads > 256 || a.parts * mean <= 32 : a.parts * most <= 64;
    const dim3 threads(four ? 256 : 1024);
    auto merge = [&](auto kernel, const auto &args) { hipLaunchKernelGGL(kernel, each, threads, 0, ctx->stream, args); };
    if (shared > 0)
      merge(four ? merge_kernel<4, SharedArgs> : merge_kernel<16, SharedArgs>, a);
    else
      merge(four ? merge_kernel<4, AttendArgs> : merge_kernel<16, AttendArgs>, alone);
    FOCR_HIP_CHECK(hipGetLastError());
  }
  return FOCR_OK;
}

}  // namespace
}  // namespace focr

using namespace focr;

extern "C" {

int focr_kv_pages_create(focr_ctx *handle, size_t n_pages, size_t page_size, size_t n_seqs, size_t seq_pages,
                         size_t n_heads, size_t n_key_heads, size_t n_kv_heads, size_t head_dim, focr_kv_pages **out) {
  Ctx *ctx = reinterpret_cast<Ctx *>(handle);
  FOCR_REQUIRE(ctx && out, FOCR_E_ARG, "focr_kv_pages_create: null argument");
  FOCR_REQUIRE(head_dim == 64, FOCR_E_UNSUPPORTED, "the paged cache takes head_dim 64");
  FOCR_REQUIRE(n_heads > 0 && n_kv_heads > 0 && n_heads % n_kv_heads == 0 && n_heads <= 1024, FOCR_E_SHAPE,
               "focr_kv_pages_create: GQA grouping");
  FOCR_REQUIRE(n_key_heads == n_kv_heads || n_key_heads == n_heads, FOCR_E_SHAPE,
               "focr_kv_pages_create: keys are held for each KV head or for each query head");
  FOCR_REQUIRE(page_size >= kBlock && page_size <= 4096 && (page_size & (page_size - 1)) == 0, FOCR_E_SHAPE,
               "focr_kv_pages_create: page_size is a power of two from 16 to 4096");
  FOCR_REQUIRE(n_pages > 0 && n_pages < (size_t(1) << 31) && n_seqs > 0 && n_seqs <= 65535 && seq_pages > 0 &&
                   seq_pages * page_size < (size_t(1) << 30) && seq_pages < (size_t(1) << 30),
               FOCR_E_SHAPE, "focr_kv_pages_create: sizes");
  FOCR_HIP_CHECK(hipSetDevice(ctx->device));
  Pages *kv = new (std::nothrow) Pages();
  FOCR_REQUIRE(kv, FOCR_E_ARG, "focr_kv_pages_create: out of host memory");
  kv->device = ctx->device;
  kv->n_pages = n_pages;
  kv->page = page_size;
  kv->n_seqs = n_seqs;
  kv->seq_pages = seq_pages;
  kv->n_heads = n_heads;
  kv->key_heads = n_key_heads;
  kv->kv_heads = n_kv_heads;
  for (size_t b = page_size / kBlock; b > 1; b /= 2) kv->shift++;
  const size_t blocks = n_pages * (page_size / kBlock), heads = n_key_heads + n_kv_heads;
  struct {
    void **at;
    size_t bytes;
    int32_t value;
  } buffers[] = {{reinterpret_cast<void **>(&kv->k_codes), blocks * n_key_heads * kBlockBytes, 0},
                 {reinterpret_cast<void **>(&kv->v_codes), blocks * n_kv_heads * kBlockBytes, 0},
                 {reinterpret_cast<void **>(&kv->k_scales), blocks * n_key_heads * sizeof(float), 0},
                 {reinterpret_cast<void **>(&kv->v_scales), blocks * n_kv_heads * sizeof(float), 0},
                 {reinterpret_cast<void **>(&kv->k_writers), blocks * n_key_heads * sizeof(int32_t), -1},
                 {reinterpret_cast<void **>(&kv->v_writers), blocks * n_kv_heads * sizeof(int32_t), -1},
                 {reinterpret_cast<void **>(&kv->table), n_seqs * seq_pages * sizeof(int32_t), -1},
                 {reinterpret_cast<void **>(&kv->open), n_seqs * heads * 2 * kBlock * 64 * sizeof(float), 0},
                 {reinterpret_cast<void **>(&kv->tags), n_seqs * heads * 2 * sizeof(int32_t), -1},
                 {reinterpret_cast<void **>(&kv->refused), n_seqs * sizeof(int32_t), 0}};
  for (auto &b : buffers) {
    hipError_t err = hipMalloc(b.at, b.bytes);
    if (err == hipSuccess) {
      kv->device_bytes += b.bytes;
      hipLaunchKernelGGL(fill_kernel, dim3(1024), dim3(256), 0, ctx->stream, static_cast<int32_t *>(*b.at),
                         b.bytes / sizeof(int32_t), b.value);
      err = hipGetLastError();
    }
    if (err != hipSuccess) {
      (void)hipStreamSynchronize(ctx->stream);
      free_pages(kv);
      delete kv;
      return set_error(FOCR_E_HIP, std::string("focr_kv_pages_create: ") + hipGetErrorString(err));
    }
  }
  // The cache may be used on another stream next.
  const hipError_t err = hipStreamSynchronize(ctx->stream);
  if (err != hipSuccess) {
    free_pages(kv);
    delete kv;
    return set_error(FOCR_E_HIP, std::string("focr_kv_pages_create: ") + hipGetErrorString(err));
  }
  *out = reinterpret_cast<focr_kv_pages *>(kv);
  return FOCR_OK;
}

int focr_kv_pages_free(focr_kv_pages *handle) {
  Pages *kv = reinterpret_cast<Pages *>(handle);
  if (!kv) return FOCR_OK;
  free_pages(kv);
  delete kv;
  return FOCR_OK;
}

int focr_kv_pages_info(const focr_kv_pages *handle, size_t *n_pages, size_t *page_size, size_t *n_seqs,
                       size_t *seq_pages, size_t *device_bytes) {
  const Pages *kv = reinterpret_cast<const Pages *>(handle);
  FOCR_REQUIRE(kv, FOCR_E_ARG, "focr_kv_pages_info: null cache");
  if (n_pages) *n_pages = kv->n_pages;
  if (page_size) *page_size = kv->page;
  if (n_seqs) *n_seqs = kv->n_seqs;
  if (seq_pages) *seq_pages = kv->seq_pages;
  if (device_bytes) *device_bytes = kv->device_bytes;
  return FOCR_OK;
}

int focr_kv_pages_map(focr_ctx *handle, focr_kv_pages *pages, size_t seq, size_t first, size_t count,
                      const int32_t *ids) {
  Ctx *ctx = reinterpret_cast<Ctx *>(handle);
  Pages *kv = reinterpret_cast<Pages *>(pages);
  FOCR_REQUIRE(ctx && kv, FOCR_E_ARG, "focr_kv_pages_map: null argument");
  FOCR_REQUIRE(kv->device == ctx->device, FOCR_E_ARG, "focr_kv_pages_map: the cache is on another device than the context");
  FOCR_REQUIRE(seq < kv->n_seqs && first <= kv->seq_pages && count <= kv->seq_pages - first, FOCR_E_SHAPE,
               "focr_kv_pages_map: outside the sequence's pages");
  if (count == 0) return FOCR_OK;
  FOCR_REQUIRE(ids, FOCR_E_ARG, "focr_kv_pages_map: null pages");
  for (size_t i = 0; i < count; i++)
    FOCR_REQUIRE(ids[i] >= -1 && ids[i] < static_cast<int64_t>(kv->n_pages), FOCR_E_VALUE, "focr_kv_pages_map: no such page");
  FOCR_HIP_CHECK(hipSetDevice(ctx->device));
  const size_t heads = kv->key_heads + kv->kv_heads;
  for (size_t at = 0; at < count; at += kMapped) {
    MapArgs a = {};
    a.table = kv->table + seq * kv->seq_pages;
    a.tags = kv->tags + seq * heads * 2;
    a.first = static_cast<int>(first + at);
    a.count = static_cast<int>(count - at < kMapped ? count - at : kMapped);
    a.shift = kv->shift;
    a.heads = static_cast<int>(heads);
    for (int i = 0; i < a.count; i++) a.pages[i] = ids[at + i];
    hipLaunchKernelGGL(map_kernel, dim3(1), dim3(256), 0, ctx->stream, a);
    FOCR_HIP_CHECK(hipGetLastError());
  }
  return FOCR_OK;
}

int focr_kv_pages_append(focr_ctx *handle, focr_kv_pages *pages, const float *k, const float *v, size_t rows,
                         const int32_t *row_start, const int32_t *lens, size_t n_seqs) {
  Ctx *ctx = reinterpret_cast<Ctx *>(handle);
  Pages *kv = reinterpret_cast<Pages *>(pages);
  const int rc = check_batch("focr_kv_pages_append", ctx, kv, rows, row_start, lens, n_seqs);
  if (rc != FOCR_OK || rows == 0 || n_seqs == 0) return rc;
  FOCR_REQUIRE(k && v, FOCR_E_ARG, "focr_kv_pages_append: null buffer");
  AppendArgs a = {};
  a.c = cache_of(kv, rows, row_start, lens, n_seqs);
  a.k = k;
  a.v = v;
  return launch_append(ctx, a, false);
}

int focr_kv_pages_qkv_rows(focr_ctx *handle, focr_kv_pages *pages, const float *qkv, size_t rows, const float *rope,
                           const int32_t *row_start, const int32_t *lens, size_t n_seqs, float *q) {
  Ctx *ctx = reinterpret_cast<Ctx *>(handle);
  Pages *kv = reinterpret_cast<Pages *>(pages);
  const int rc = check_batch("focr_kv_pages_qkv_rows", ctx, kv, rows, row_start, lens, n_seqs);
  if (rc != FOCR_OK || rows == 0 || n_seqs == 0) return rc;
  FOCR_REQUIRE(qkv && rope && q, FOCR_E_ARG, "focr_kv_pages_qkv_rows: null buffer");
  AppendArgs a = {};
  a.c = cache_of(kv, rows, row_start, lens, n_seqs);
  a.qkv = qkv;
  a.rope = rope;
  a.q = q;
  return launch_append(ctx, a, true);
}

int focr_kv_pages_qkv_rows_at(focr_ctx *handle, focr_kv_pages *pages, const float *qkv, size_t rows,
                              const float *positions, size_t axes, const float *frequencies, const int32_t *row_start,
                              const int32_t *lens, size_t n_seqs, float *q) {
  Ctx *ctx = reinterpret_cast<Ctx *>(handle);
  Pages *kv = reinterpret_cast<Pages *>(pages);
  const int rc = check_batch("focr_kv_pages_qkv_rows_at", ctx, kv, rows, row_start, lens, n_seqs);
  if (rc != FOCR_OK) return rc;
  FOCR_REQUIRE(axes >= 1 && axes <= kMaxAxes, FOCR_E_SHAPE, "focr_kv_pages_qkv_rows_at: 1 to 4 axes");
  if (rows == 0 || n_seqs == 0) return FOCR_OK;
  FOCR_REQUIRE(qkv && positions && frequencies && q, FOCR_E_ARG, "focr_kv_pages_qkv_rows_at: null buffer");
  FOCR_REQUIRE(reinterpret_cast<uintptr_t>(frequencies) % 8 == 0, FOCR_E_ARG,
               "focr_kv_pages_qkv_rows_at: frequencies stand on 8 bytes");
  AppendArgs a = {};
  a.c = cache_of(kv, rows, row_start, lens, n_seqs);
  a.qkv = qkv;
  a.positions = positions;
  a.frequencies = frequencies;
  a.axes = static_cast<int>(axes);
  a.q = q;
  return launch_append(ctx, a, true);
}

int focr_kv_pages_attention(focr_ctx *handle, const focr_kv_pages *pages, const float *q, size_t rows,
                            const int32_t *row_start, const int32_t *lens, size_t n_seqs, size_t max_len,
                            const float *sinks, float *out) {
  return launch_attend("focr_kv_pages_attention", reinterpret_cast<Ctx *>(handle), reinterpret_cast<const Pages *>(pages), q,
                       rows, row_start, lens, n_seqs, max_len, 0, 0, sinks, out);
}

int focr_kv_pages_attention_shared(focr_ctx *handle, const focr_kv_pages *pages, const float *q, size_t rows,
                                   const int32_t *row_start, const int32_t *lens, size_t n_seqs, size_t max_len,
                                   size_t prefix_seq, size_t shared_len, const float *sinks, float *out) {
  return launch_attend("focr_kv_pages_attention_shared", reinterpret_cast<Ctx *>(handle),
                       reinterpret_cast<const Pages *>(pages), q, rows, row_start, lens, n_seqs, max_len, prefix_seq,
                       shared_len, sinks, out);
}

int focr_kv_pages_dequantize(focr_ctx *handle, const focr_kv_pages *pages, size_t rows, const int32_t *row_start,
                             const int32_t *lens, size_t n_seqs, float *k, float *v) {
  Ctx *ctx = reinterpret_cast<Ctx *>(handle);
  const Pages *kv = reinterpret_cast<const Pages *>(pages);
  const int rc = check_batch("focr_kv_pages_dequantize", ctx, kv, rows, row_start, lens, n_seqs);
  if (rc != FOCR_OK || rows == 0 || n_seqs == 0) return rc;
  FOCR_REQUIRE(k && v, FOCR_E_ARG, "focr_kv_pages_dequantize: null buffer");
  const Cache c = cache_of(kv, rows, row_start, lens, n_seqs);
  // n rows touch at most (n + 14) / 16 + 1 blocks.
  const size_t units = row_start ? rows / kBlock + 2 * (rows < n_seqs ? rows : n_seqs) : n_seqs;
  FOCR_HIP_CHECK(hipSetDevice(ctx->device));
  hipLaunchKernelGGL(read_kernel, dim3(static_cast<unsigned>(units), static_cast<unsigned>((c.key_heads + c.kv_heads + 3) / 4)),
                     dim3(256), 0, ctx->stream, c, k, v);
  FOCR_HIP_CHECK(hipGetLastError());
  return FOCR_OK;
}

int focr_kv_pages_refused(focr_ctx *handle, focr_kv_pages *pages, int32_t *seqs) {
  Ctx *ctx = reinterpret_cast<Ctx *>(handle);
  Pages *kv = reinterpret_cast<Pages *>(pages);
  FOCR_REQUIRE(ctx && kv && seqs, FOCR_E_ARG, "focr_kv_pages_refused: null argument");
  FOCR_REQUIRE(kv->device == ctx->device, FOCR_E_ARG, "focr_kv_pages_refused: the cache is on another device than the context");
  FOCR_HIP_CHECK(hipSetDevice(ctx->device));
  FOCR_HIP_CHECK(hipMemcpyAsync(seqs, kv->refused, kv->n_seqs * sizeof(int32_t), hipMemcpyDeviceToHost, ctx->stream));
  hipLaunchKernelGGL(fill_kernel, dim3(1), dim3(256), 0, ctx->stream, kv->refused, kv->n_seqs, 0);
  FOCR_HIP_CHECK(hipGetLastError());
  FOCR_HIP_CHECK(hipStreamSynchronize(ctx->stream));
  return FOCR_OK;
}

}  // extern "C"
