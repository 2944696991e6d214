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
__device__ __forceinline__ void norm_rotate(v4f (&x)[4], const v4f (&f)[4]) {
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
  const float scales = __fdiv_rn(1.0f, __builtin_sqrtf(__fdiv_rn(sums, 64.0f) + 1.1920929e-7f));
  const float scale[4] = {row_lane<0>(scales), row_lane<1>(scales), row_lane<2>(scales), row_lane<3>(scales)};
#pragma unroll
  for (int s = 0; s < 4; s++) {
    const v4f y = {x[s][0] * scale[s], x[s][1] * scale[s], x[s][2] * scale[s], x[s][3] * scale[s]};
    x[s] = v4f{y[0] * f[s][0] - y[1] * f[s][1], y[0] * f[s][1] + y[1] * f[s][0], y[2] * f[s][2] - y[3] * f[s][3],
               y[2] * f[s][3] + y[3] * f[s][2]};
  }
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

// A sequence's rows for attention; false where there is nothing to do (n = 0) or it
// is refused (bad), but for what `overlaps` says.
__device__ __forceinline__ bool attend_span(const AttendArgs &a, int seq, int &len, int &first, int &n, bool &bad) {
  bad = !a.c.span(seq, len, first, n);
  if (n > 8 || (n > 0 && len + n > a.max_len)) bad = true;
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
template <bool WIDE>
__global__ __launch_bounds__(256, 3) void attend_kernel(AttendArgs a) {
  const Cache &c = a.c;
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Workgroups go to the 8 XCDs in turn: those of the key heads of one value head
  // follow one another on the same one, whose L2 then holds the values for all.
  const int share = c.key_heads / c.kv_heads, turn_of = blockIdx.x / 8;
  int task = (turn_of / share * 8 + blockIdx.x % 8) * share + turn_of % share;
  const int key_head = task % c.key_heads;
  task /= c.key_heads;
  const int tile = task % a.tiles;
  task /= a.tiles;
  const int part = task % a.parts, seq = task / a.parts;
  if (seq >= c.n_seqs) return;
  const int group = c.n_heads / c.key_heads, value_head = key_head * c.kv_heads / c.key_heads;
  int len, first, n;
  bool bad;
  const int start = start_of(c, seq);
  if (!attend_span(a, seq, len, first, n, bad)) {
    if (bad && a.parts == 1 && tile == 0 && wave == 0) refuse_rows(a, seq, key_head * group, group);
    return;
  }
  const int limit = len + n, from_key = part * a.chunk;
  if (16 * tile >= group * n || from_key >= limit) return;
  // Waves: runs of the part's keys, in whole 64s, times quads of columns.
  const int columns = group * n, left = columns - 16 * tile;
  const int quads = left <= 4 ? 1 : left <= 8 ? 2 : 4, runs = 4 / quads, run = wave / quads, quad = wave % quads;
  const int to_key = from_key + a.chunk < limit ? from_key + a.chunk : limit;
  const int each = (to_key - from_key + 64 * runs - 1) / (64 * runs) * 64;
  const int begin = from_key + run * each, end = begin + each < to_key ? begin + each : to_key;
  const int column0 = 16 * tile + 4 * quad;

  // 64 keys: lane's key block is l16 / 4 of four, its value block g. In a page of 64
  // positions or more (WIDE) they follow one another, and their addresses are scalar
  // but for the lane's share; otherwise each lane looks its blocks' pages up (past the
  // last block, that one again). A block without a page is NaN.
  const int last_block = (limit - 1) / kBlock, blocks_mask = (1 << c.shift) - 1;
  const int32_t *table = c.table + static_cast<size_t>(seq) * c.seq_pages;
  typedef __attribute__((address_space(4))) const int32_t scalar_table;  // read by scalar loads
  bool missing = false;
  struct Found {
    int k_page, v_page;
  };
  auto find = [&](int key0) {
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
  };
  const int k_lane = l16 % 4 * 64 + g * 16, v_lane = l16 * 16;
  auto load = [&](const Found &f, int key0, Stage &s) {
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
  };
  Found next;
  Stage stage[2];
  const bool works = begin < end && column0 < columns;
  if (works) next = find(begin);

  // Column column0 + q: query row first + column % n, head key_head * group +
  // column / n. Lane l16 brings row l16 of the first product (query l16 / 4, byte
  // l16 % 4), lane (l16, g) works on query g.
  v4i digit;
  float q_factor;
  int visible;
  if (works) {
    float4 x[4];
    const int wanted = column0 + l16 / 4, column = wanted < columns ? wanted : columns - 1;
    const float *q = a.q + (static_cast<size_t>(first + column % n) * c.n_heads + key_head * group + column / n) * 64 + 16 * g;
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = reinterpret_cast<const float4 *>(q)[i];
    load(next, begin, stage[0]);
    next = find(begin + 64);
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
    const float factor = finite ? __builtin_ldexpf(0.180336880111120426f, e - 30) : __builtin_nanf("");
    q_factor = __int_as_float(__builtin_amdgcn_ds_bpermute(4 * (4 * g), __float_as_int(factor)));
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
    const int mine = column0 + g;
    visible = len + (mine < columns ? mine : columns - 1) % n + 1;
  }
  const float ninf = -__builtin_inff();
  float m = ninf, den = 0.0f;
  int power = -300;  // 2^power above every block scale of the values so far
  v4f acc[4];
#pragma unroll
  for (int d = 0; d < 4; d++) acc[d] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  // The parts of the weights: [column 4 d + q][64 keys], a wave's own. Rows of 72, so
  // that 16 columns' 16 bytes lie in different banks; there is no fourth part.
  constexpr int kTurned = 72;
  __shared__ __attribute__((aligned(16))) uint16_t turned[4][16 * kTurned];
  uint16_t *const turn_to = turned[wave] + g * kTurned + 4 * l16;
  const uint16_t *const turn_from = turned[wave] + l16 * kTurned + 16 * g;
  *reinterpret_cast<uint2 *>(turn_to + 12 * kTurned) = make_uint2(0, 0);

  // The sums times `scaled` of query g: column 4 d + q's lanes take that of query q.
  auto rescale = [&](float scaled) {
    const float s0 = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(scaled), 0));
    const float s1 = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(scaled), 16));
    const float s2 = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(scaled), 32));
    const float s3 = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(scaled), 48));
    const float f = l16 & 2 ? (l16 & 1 ? s3 : s2) : (l16 & 1 ? s1 : s0);
#pragma unroll
    for (int d = 0; d < 4; d++)
#pragma unroll
      for (int i = 0; i < 4; i++) acc[d][i] = acc[d][i] * f;
  };

  // Two FP32 numbers' upper halves, the first one's low.
  auto upper = [](uint32_t second, uint32_t first) { return __builtin_amdgcn_perm(second, first, 0x07060302u); };
  auto as_bf = [](uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    const v4i words = {static_cast<int>(a), static_cast<int>(b), static_cast<int>(c), static_cast<int>(d)};
    return __builtin_bit_cast(v8bf, words);
  };
  // Eight codes as BF16 numbers.
  auto codes_of = [&](int first, int second) {
    const uint32_t w[2] = {static_cast<uint32_t>(first), static_cast<uint32_t>(second)};
    uint32_t to[4];
#pragma unroll
    for (int i = 0; i < 2; i++) {
      to[2 * i] = upper(__float_as_uint(sdwa_cvt<1>(w[i])), __float_as_uint(sdwa_cvt<0>(w[i])));
      to[2 * i + 1] = upper(__float_as_uint(sdwa_cvt<3>(w[i])), __float_as_uint(sdwa_cvt<2>(w[i])));
    }
    return as_bf(to[0], to[1], to[2], to[3]);
  };

  auto consume = [&](const Stage &s, int key0) {
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
    float p[4];
    const float factor = q_factor * k_scale;
#pragma unroll
    for (int t = 0; t < 4; t++) {
      const v4i zero = {0, 0, 0, 0};
      const v4i dots = __builtin_amdgcn_mfma_i32_16x16x64_i8(digit, s.k[t], zero, 0, 0, 0);
      // A sum is below 2^20, so two of them fit 32 bits.
      const float sum = fmaf_(static_cast<float>((dots[3] << 8) + dots[2]), 65536.0f, static_cast<float>((dots[1] << 8) + dots[0]));
      p[t] = sum * factor;
      if (key0 + 4 * l16 + t >= visible) p[t] = ninf;
    }
    float top = __builtin_fmaxf(__builtin_fmaxf(p[0], p[1]), __builtin_fmaxf(p[2], p[3]));
    top = __builtin_fmaxf(m, row_max(top));
    const float from = top == ninf ? 0.0f : top;
    if (__any(top > m) || lower < 0) {
      const float keep = __builtin_amdgcn_exp2f(m - from);
      den = den * keep;
      rescale(__builtin_ldexpf(keep, lower));
      m = top;
    }
    uint32_t part[3][4];
#pragma unroll
    for (int t = 0; t < 4; t++) {
      const float e = __builtin_amdgcn_exp2f(p[t] - from);
      den = den + e;
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
      acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(codes_of(s.v[d][0], s.v[d][1]), low, acc[d], 0, 0, 0);
      acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(codes_of(s.v[d][2], s.v[d][3]), high, acc[d], 0, 0, 0);
    }
  };
  // While one 64 keys are worked on, the next are on their way, and before them the
  // pages of those after: no load is under a branch, so the waits count what is
  // still out.
  auto turn = [&](const Stage &now, Stage &then, int key0, auto more) {
    if constexpr (decltype(more)::value) {
      const Found after = find(key0 + 128);
      load(next, key0 + 64, then);
      next = after;
    }
    consume(now, key0);
  };
  if (works) {
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
  if (__any(missing) && lane == 0) c.refused[seq] = 1;
  // Asked here, where no load is waited for.
  if (overlaps(c, seq, first, start)) {
    if (a.parts == 1 && tile == 0 && wave == 0) refuse_rows(a, seq, key_head * group, group);
    return;
  }

  // The waves' states meet in LDS: [run][column], 16 in all.
  __shared__ float s_m[16], s_den[16];
  __shared__ __attribute__((aligned(16))) float s_o[16][68];
  den = den + row_ror<8>(den);
  den = den + row_ror<4>(den);
  den = den + row_ror<2>(den);
  den = den + row_ror<1>(den);
  if (l16 == 0) {
    s_m[4 * wave + g] = m;
    s_den[4 * wave + g] = den;
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
    if (l16 < 4) *reinterpret_cast<v4f *>(&s_o[4 * wave + l16][16 * d + 4 * g]) = o;
  }
  __syncthreads();
  // Thread: a column and four dims.
  const int col = threadIdx.x / 16, dim = threadIdx.x % 16 * 4, wide = 4 * quads;
  const int out_column = 16 * tile + col;
  if (col >= wide || out_column >= columns) return;
  float top = s_m[col], total = 0.0f;
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
  const int out_head = key_head * group + out_column / n;
  const size_t out_row = static_cast<size_t>(first + out_column % n) * c.n_heads + out_head;
  if (a.parts == 1) {
    const float factor = sink_factor(a.sinks, out_head, top, total);
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] = __fdiv_rn(o[i], total) * factor;
    *reinterpret_cast<v4f *>(a.out + out_row * 64 + dim) = o;
    return;
  }
  const size_t at = out_row * a.parts + part;
  *reinterpret_cast<v4f *>(a.part_o + at * 64 + dim) = o;
  if (dim == 0) *reinterpret_cast<float2 *>(a.part_md + at * 2) = make_float2(top, total);
}

// The parts of a sequence's rows of one head: as many of the waves for each row as
// there are, lane = element, eight parts of a wave in flight. Bound by the launch and
// the trips to memory: 4.4 us for 7 parts of 25 rows, 5.3 for 57 parts of two.
template <int WAVES>
__global__ __launch_bounds__(64 * WAVES) void merge_kernel(AttendArgs a) {
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
  const int parts = (len + n - 1) / a.chunk + 1;
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
  const int heads = c.key_heads + c.kv_heads + (qkv ? c.n_heads : 0);
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
  if (qkv)
    hipLaunchKernelGGL(append_kernel<true>, grid, dim3(256), 0, ctx->stream, a);
  else
    hipLaunchKernelGGL(append_kernel<false>, grid, dim3(256), 0, ctx->stream, a);
  FOCR_HIP_CHECK(hipGetLastError());
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

int focr_kv_pages_attention(focr_ctx *handle, const focr_kv_pages *pages, const float *q, size_t rows,
                            const int32_t *row_start, const int32_t *lens, size_t n_seqs, size_t max_len,
                            const float *sinks, float *out) {
  Ctx *ctx = reinterpret_cast<Ctx *>(handle);
  const Pages *kv = reinterpret_cast<const Pages *>(pages);
  int rc = check_batch("focr_kv_pages_attention", ctx, kv, rows, row_start, lens, n_seqs);
  if (rc != FOCR_OK || rows == 0 || n_seqs == 0) return rc;
  FOCR_REQUIRE(q && out, FOCR_E_ARG, "focr_kv_pages_attention: null buffer");
  FOCR_REQUIRE(max_len > 0 && max_len <= kv->seq_pages * kv->page, FOCR_E_SHAPE,
               "focr_kv_pages_attention: max_len is 1 .. what a sequence's pages hold");
  AttendArgs a = {};
  a.c = cache_of(kv, rows, row_start, lens, n_seqs);
  a.q = q;
  a.sinks = sinks;
  a.out = out;
  a.max_len = static_cast<int>(max_len);
  const size_t most = row_start ? std::min<size_t>(rows, 8) : 1;
  const size_t group = kv->n_heads / kv->key_heads;
  a.tiles = static_cast<int>((group * most + 15) / 16);
  // Parts of whole 256 keys, at most 4,096 up to a million positions. Few sequences
  // need only fill the chip (us a call with 512 / 1,024 / 2,048 workgroups: one of
  // 131,072 positions 32.9 / 36.8 / 37.7, four of up to 16,000 16.3 / 17.8 / 18.8; six of
  // up to 3,000 with up to 8 rows 17.6 / 15.4 / 15.9); more, of different lengths, want
  // parts to spare (20 of up to 9,000 49.0 / 47.1 / 44.7, 40 of up to 5,000 with up to 8
  // rows 84.7 / 84.8 / 63.7).
  const size_t heads = n_seqs * kv->key_heads * a.tiles;
  const size_t enough = n_seqs <= 2 ? 512 : n_seqs <= 8 ? 1024 : 2048;
  const size_t want = heads >= enough ? 1 : enough / heads;
  const size_t chunk = std::max(std::min<size_t>((max_len + want - 1) / want, 4096), (max_len + kMaxParts - 1) / kMaxParts);
  a.chunk = static_cast<int>((chunk + 255) / 256 * 256);
  a.parts = static_cast<int>((max_len + a.chunk - 1) / a.chunk);
  const size_t share = kv->key_heads / kv->kv_heads;
  const size_t grid = (heads * a.parts + 8 * share - 1) / (8 * share) * (8 * share);
  FOCR_REQUIRE(grid < (size_t(1) << 31), FOCR_E_SHAPE, "focr_kv_pages_attention: too many sequences and heads");
  const size_t slots = rows * kv->n_heads * a.parts;
  FOCR_HIP_CHECK(hipSetDevice(ctx->device));
  if (a.parts > 1) {
    rc = ensure_scratch(ctx, slots * 66 * sizeof(float));
    if (rc != FOCR_OK) return rc;
    a.part_o = static_cast<float *>(ctx->scratch);
    a.part_md = a.part_o + slots * 64;
  }
  if (kv->page >= 64)
    hipLaunchKernelGGL(attend_kernel<true>, dim3(static_cast<unsigned>(grid)), dim3(256), 0, ctx->stream, a);
  else
    hipLaunchKernelGGL(attend_kernel<false>, dim3(static_cast<unsigned>(grid)), dim3(256), 0, ctx->stream, a);
  FOCR_HIP_CHECK(hipGetLastError());
  if (a.parts > 1) {
    const dim3 each(static_cast<unsigned>(kv->n_heads), static_cast<unsigned>(n_seqs));
    // Parts of all a sequence's rows (us a call with 4 / 16 waves: 26 parts of one row
    // 9.8 / 10.4, 3 of one in 64 sequences 112 / 120; 57 of two 34.8 / 32.8, 59 of
    // eight 33.3 / 20.3).
    if (a.parts * most <= 64)
      hipLaunchKernelGGL(merge_kernel<4>, each, dim3(256), 0, ctx->stream, a);
    else
      hipLaunchKernelGGL(merge_kernel<16>, each, dim3(1024), 0, ctx->stream, a);
    FOCR_HIP_CHECK(hipGetLastError());
  }
  return FOCR_OK;
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
