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
// Key codes stand as [position][64], signed; value codes as [dim][16 positions],
// plus 128: both what the attention's matrix instructions take 16 bytes at a time.
//
// A block that is not full is written again by the next append, with the scale that
// its positions then need. So that this rounds every value once, the last two
// blocks of a sequence are also kept in FP32 beside the pages (two, so that a step
// that takes back up to 16 positions finds them too): what the cache holds depends
// on the rows appended, and not on how many at a time. Where a block is not
// there (a sequence that goes on from pages it was given, or goes back further),
// its earlier positions are taken from its codes.
#include <algorithm>
#include <new>
#include <type_traits>

#include "decode_common.hpp"
#include "rms_tree.hpp"

namespace focr {
namespace {

constexpr int kBlock = 16, kBlockBytes = kBlock * 64;

typedef int v4i __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

struct Pages {
  int device = 0, shift = 0;  // log2 of the blocks of a page
  size_t n_pages = 0, page = 0, n_seqs = 0, seq_pages = 0, n_heads = 0, key_heads = 0, kv_heads = 0;
  int8_t *k_codes = nullptr;   // [page][key head][block][1 KB]
  uint8_t *v_codes = nullptr;  // [page][KV head][block][1 KB]
  float *k_scales = nullptr, *v_scales = nullptr;  // [page][head][block]
  int32_t *table = nullptr;    // [sequence][seq_pages], -1: no page
  float *open = nullptr;       // [sequence][key heads, then KV heads][block % 2][16][64]
  int32_t *tags = nullptr;     // [sequence][heads][2]: the block that `open` holds, or -1
  int32_t *refused = nullptr;  // [sequence]
  size_t device_bytes = 0;
};

// What the kernels read of a cache, and a call's rows.
struct Cache {
  int8_t *k_codes;
  uint8_t *v_codes;
  float *k_scales, *v_scales;
  const int32_t *table;
  float *open;
  int32_t *tags, *refused;
  int shift, seq_pages, n_pages, n_heads, key_heads, kv_heads;
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

// decode::norm_rope, bit for bit, without LDS: lane = element.
__device__ __forceinline__ float norm_rotate(float x, float2 factor, int lane) {
  const float leaf = fold_leaf_pair(x * x);
  const float leaf0 = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(leaf), 0));
  const float leaf1 = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(leaf), 32));
  const float scale = __fdiv_rn(1.0f, __builtin_sqrtf(__fdiv_rn(leaf0 + leaf1, 64.0f) + 1.1920929e-7f));
  const float y = x * scale;
  const float partner = rms_dpp<0xB1>(y);
  const bool even = (lane & 1) == 0;
  const float a = even ? y : partner, b = even ? partner : y;
  return even ? a * factor.x - b * factor.y : a * factor.y + b * factor.x;
}

// Units of an append: the blocks of a sequence's rows, the first and the last two
// together (they read and write the FP32 blocks), the others one by one.
__device__ __forceinline__ int touched(int len, int n) { return (len + n - 1) / kBlock - len / kBlock + 1; }

// A wave takes one unit and one head: a stored head (keys, then values), or with QKV
// a query head. Lane = element; a block's 16 positions are 16 registers.
template <bool QKV>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
  const Cache &c = a.c;
  __shared__ __attribute__((aligned(16))) int8_t turn[4][kBlockBytes];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int head = blockIdx.y * 4 + wave, stored = c.key_heads + c.kv_heads;
  const auto of = [](int len, int n) {
    const int blocks = touched(len, n);
    return blocks <= 3 ? 1 : blocks - 2;
  };
  Unit unit;
  const bool found = find_unit(c, blockIdx.x, of, unit);
  if (blockIdx.x == 0 && head == 0 && c.row_start) {
    // Marks every refused sequence.
    Unit none;
    find_unit(c, 0x7fffffff, of, none);
  }
  if (!found || head >= stored + (QKV ? c.n_heads : 0)) return;
  const bool is_key = head < c.key_heads, is_query = head >= stored;
  const int qkv_width = (c.n_heads + 2 * c.kv_heads) * 64;
  // The head's element in a row, and its pair's factors.
  int from, pair = 0;
  const float *source;
  size_t width;
  if constexpr (QKV) {
    source = a.qkv;
    width = qkv_width;
    if (is_query) {
      from = (head - stored) * 64;
      pair = head - stored;
    } else if (is_key) {
      from = (c.n_heads + head * c.kv_heads / c.key_heads) * 64;
      pair = head * (c.n_heads / c.key_heads);
    } else {
      from = (c.n_heads + c.kv_heads + head - c.key_heads) * 64;
    }
  } else {
    source = is_key ? a.k : a.v;
    width = static_cast<size_t>(is_key ? c.key_heads : c.kv_heads) * 64;
    from = (is_key ? head : head - c.key_heads) * 64;
  }
  const int first_block = unit.len / kBlock, blocks = touched(unit.len, unit.n), last_block = first_block + blocks - 1;
  const int held = is_key ? c.key_heads : c.kv_heads, at_head = is_key ? head : head - c.key_heads;
  const size_t slot = (static_cast<size_t>(unit.seq) * stored + head) * 2;

  auto process = [&](int block) {
    const int row0 = block * kBlock - unit.len;  // the row of its first position
    const bool saved = block >= last_block - 1;
    if (is_query) {
      float x[kBlock];
      float2 f[kBlock];
#pragma unroll
      for (int t = 0; t < kBlock; t++) {
        const int row = row0 + t, at = unit.first + (row >= 0 && row < unit.n ? row : 0);
        x[t] = source[at * width + from + lane];
        f[t] = reinterpret_cast<const float2 *>(a.rope)[(static_cast<size_t>(at) * c.n_heads + pair) * 32 + lane / 2];
      }
#pragma unroll
      for (int t = 0; t < kBlock; t++) {
        const int row = row0 + t;
        if (row >= 0 && row < unit.n)
          a.q[(static_cast<size_t>(unit.first + row) * c.n_heads + pair) * 64 + lane] = norm_rotate(x[t], f[t], lane);
      }
      return;
    }
    const long number = c.block_at(unit.seq, block, held, at_head);
    if (number < 0) {
      c.refused[unit.seq] = 1;
      return;
    }
    float *const open = c.open + (slot + block % 2) * kBlock * 64;
    const bool kept = row0 < 0 && c.tags[slot + block % 2] == block;
    float *scale_at = (is_key ? c.k_scales : c.v_scales) + number;
    // Earlier positions from the FP32 block, new ones from the rows.
    float x[kBlock];
    float2 f[kBlock];
#pragma unroll
    for (int t = 0; t < kBlock; t++) {
      const int row = row0 + t, at = unit.first + (row >= 0 && row < unit.n ? row : 0);
      x[t] = *(row < 0 ? open + t * 64 + lane : source + at * width + from + lane);
      if (QKV && is_key)
        f[t] = reinterpret_cast<const float2 *>(a.rope)[(static_cast<size_t>(at) * c.n_heads + pair) * 32 + lane / 2];
    }
    if (row0 < 0 && !kept) {
      // From the codes.
      const float scale = *scale_at;
#pragma unroll
      for (int t = 0; t < kBlock; t++)
        if (row0 + t < 0) {
          const int code = is_key ? c.k_codes[number * kBlockBytes + t * 64 + lane]
                                  : c.v_codes[number * kBlockBytes + lane * kBlock + t] - 128;
          x[t] = static_cast<float>(code) * scale;
        }
    }
    uint32_t big = 0;
#pragma unroll
    for (int t = 0; t < kBlock; t++) {
      const int row = row0 + t;
      if (row >= unit.n) x[t] = 0.0f;
      if (QKV && is_key && row >= 0 && row < unit.n) x[t] = norm_rotate(x[t], f[t], lane);
      const uint32_t bits = __float_as_uint(x[t]) & 0x7fffffffu;
      big = bits > big ? bits : big;
    }
    big = wave_max_bits(big);
    float scale = __fdiv_rn(__uint_as_float(big), 127.0f);
    if (scale < 1.17549435e-38f) scale = 0.0f;
    const float inverse = scale > 0.0f ? __fdiv_rn(1.0f, scale) : 0.0f;
    const bool finite = big < 0x7f800000u;
    int code[kBlock];
#pragma unroll
    for (int t = 0; t < kBlock; t++) code[t] = finite ? static_cast<int>(__builtin_rintf(x[t] * inverse)) : 0;
    if (is_key) {
      // [position][64]: through LDS, 16 bytes a lane.
#pragma unroll
      for (int t = 0; t < kBlock; t++) turn[wave][t * 64 + lane] = static_cast<int8_t>(code[t]);
      __builtin_amdgcn_wave_barrier();
      const uint4 bytes = *reinterpret_cast<const uint4 *>(&turn[wave][lane * 16]);
      __builtin_amdgcn_wave_barrier();
      *reinterpret_cast<uint4 *>(c.k_codes + number * kBlockBytes + lane * 16) = bytes;
    } else {
      uint32_t word[4];
#pragma unroll
      for (int w = 0; w < 4; w++)
        word[w] = static_cast<uint32_t>(code[4 * w] + 128) | static_cast<uint32_t>(code[4 * w + 1] + 128) << 8 |
                  static_cast<uint32_t>(code[4 * w + 2] + 128) << 16 | static_cast<uint32_t>(code[4 * w + 3] + 128) << 24;
      *reinterpret_cast<uint4 *>(c.v_codes + number * kBlockBytes + lane * kBlock) = make_uint4(word[0], word[1], word[2], word[3]);
    }
    if (lane == 0) *scale_at = finite ? scale : __builtin_nanf("");
    if (saved) {
#pragma unroll
      for (int t = 0; t < kBlock; t++)
        if (row0 + t < unit.n && (row0 + t >= 0 || !kept)) open[t * 64 + lane] = x[t];
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
// A wave takes one block of a sequence's rows and one stored head.
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
  if (is_key) {
    // Lane: 16 elements of position lane / 4.
    const uint4 bytes = *reinterpret_cast<const uint4 *>(c.k_codes + at * kBlockBytes + lane * 16);
    const int row = row0 + lane / 4;
    if (row < 0 || row >= unit.n) return;
    float *to = k + (static_cast<size_t>(unit.first + row) * held + at_head) * 64 + lane % 4 * 16;
    const uint32_t word[4] = {bytes.x, bytes.y, bytes.z, bytes.w};
#pragma unroll
    for (int w = 0; w < 4; w++)
      reinterpret_cast<float4 *>(to)[w] = make_float4(sdwa_cvt<0>(word[w]) * scale, sdwa_cvt<1>(word[w]) * scale,
                                                      sdwa_cvt<2>(word[w]) * scale, sdwa_cvt<3>(word[w]) * scale);
    return;
  }
  // Lane: element `lane` of all 16 positions.
  const uint4 bytes = *reinterpret_cast<const uint4 *>(c.v_codes + at * kBlockBytes + lane * kBlock);
  const uint32_t word[4] = {bytes.x, bytes.y, bytes.z, bytes.w};
#pragma unroll
  for (int t = 0; t < kBlock; t++) {
    const int row = row0 + t;
    if (row >= 0 && row < unit.n)
      v[(static_cast<size_t>(unit.first + row) * held + at_head) * 64 + lane] =
          static_cast<float>(static_cast<int>((word[t / 4] >> (8 * (t % 4))) & 255) - 128) * scale;
  }
}

// ---- attention -----------------------------------------------------------------
struct AttendArgs {
  Cache c;
  const float *q, *sinks;
  float *out;
  float *part_o, *part_md;  // [row][head][part][64], [..][2]
  int max_len, chunk, parts, tiles, most;  // most: rows of a sequence at most
};

// A sequence's rows for attention; false where there is nothing to do (n = 0) or it
// is refused (bad).
__device__ __forceinline__ bool attend_span(const AttendArgs &a, int seq, int &len, int &first, int &n, bool &bad) {
  bad = !a.c.span(seq, len, first, n);
  if (n > 8 || (n > 0 && len + n > a.max_len)) bad = true;
  return n > 0 && !bad;
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

// The rows of a refused sequence, where they are rows of the call: NaN.
__device__ __forceinline__ void refuse_rows(const AttendArgs &a, int seq, int head0, int heads) {
  const Cache &c = a.c;
  const int lane = threadIdx.x & 63;
  const int begin = c.row_start ? c.row_start[seq] : seq, end = c.row_start ? c.row_start[seq + 1] : seq + 1;
  if (lane == 0) c.refused[seq] = 1;
  if (begin < 0 || end > c.rows) return;
  for (int row = begin; row < end; row++)
    for (int h = head0; h < head0 + heads; h++)
      a.out[(static_cast<size_t>(row) * c.n_heads + h) * 64 + lane] = __builtin_nanf("");
}

// The largest (sum) of lanes l, l + 16, l + 32, l + 48, in each of them.
__device__ __forceinline__ float across_max(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __builtin_fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __builtin_fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float across_sum(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// A wave takes one sequence, one key head's queries (its query heads times the
// sequence's rows, 16 at a time: the columns of both products) and one part of the
// keys, 64 at a time: four blocks, block g the business of lanes 16 g .. + 15.
//
// Scores: the query row is written as integers i 2^(e - 22) of three signed bytes
// (2^e above its largest element, so to 2^-22 of it), and the INT8 matrix instruction
// forms 16 keys' exact sums with each byte from the codes as they stand. Row
// 4 g + i of key tile t is key 16 g + 4 t + i, so that the scores of lane group g are
// those of block g, in the order in which the second product takes its keys.
// Values: codes become FP16 integers exactly (byte b under the exponent of 1024 is
// 1024 + b), and a weight times its block's scale, to a common power of two, an FP16
// pair hi + lo, together to 2^-21 of it: two FP32-accumulating products. The running
// maximum and sum are per column; the power of two is the largest block scale's so far.
struct Stage {
  v4i k[4];
  v4u v[4];
  float k_scale, v_scale;
};
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
  if (!attend_span(a, seq, len, first, n, bad)) {
    if (bad && a.parts == 1 && tile == 0 && wave == 0) refuse_rows(a, seq, key_head * group, group);
    return;
  }
  const int limit = len + n, from_key = part * a.chunk;
  if (16 * tile >= group * n || from_key >= limit) return;
  // The part's keys, in whole 64s, over the four waves.
  const int to_key = from_key + a.chunk < limit ? from_key + a.chunk : limit;
  const int each = (to_key - from_key + 255) / 256 * 64;
  const int begin = from_key + wave * each, end = begin + each < to_key ? begin + each : to_key;

  // Pages and blocks of 64 keys: lane's key block and value block (past the last
  // block, that one again: masked).
  const int last_block = (limit - 1) / kBlock, blocks_mask = (1 << c.shift) - 1;
  const int32_t *table = c.table + static_cast<size_t>(seq) * c.seq_pages;
  struct Pages64 {
    int k_block, v_block, k_page, v_page;
  };
  auto find = [&](int key0) {
    Pages64 p;
    const int b = key0 / kBlock;
    p.k_block = b + l16 / 4 < last_block ? b + l16 / 4 : last_block;
    p.v_block = b + g < last_block ? b + g : last_block;
    p.k_page = table[p.k_block >> c.shift];
    p.v_page = table[p.v_block >> c.shift];
    return p;
  };
  bool missing = false;
  auto load = [&](const Pages64 &p, Stage &s) {
    // A block without a page is NaN.
    missing |= p.v_page < 0;
    const long kp = p.k_page < 0 ? 0 : p.k_page, vp = p.v_page < 0 ? 0 : p.v_page;
    const long kn = ((kp * c.key_heads + key_head) << c.shift) + (p.k_block & blocks_mask);
    const long sn = ((vp * c.key_heads + key_head) << c.shift) + (p.v_block & blocks_mask);
    const long vn = ((vp * c.kv_heads + value_head) << c.shift) + (p.v_block & blocks_mask);
    const int8_t *k = c.k_codes + kn * kBlockBytes + l16 % 4 * 64 + g * 16;
    const uint8_t *v = c.v_codes + vn * kBlockBytes + l16 * 16;
#pragma unroll
    for (int t = 0; t < 4; t++) s.k[t] = *reinterpret_cast<const v4i *>(k + t * 256);
#pragma unroll
    for (int d = 0; d < 4; d++) s.v[d] = *reinterpret_cast<const v4u *>(v + d * 256);
    s.k_scale = c.k_scales[sn];
    s.v_scale = c.v_scales[vn];
    if (p.v_page < 0) s.k_scale = s.v_scale = __builtin_nanf("");
  };

  // This lane's column: query row first + r, head key_head * group + column / n.
  int column = 16 * tile + l16;
  const bool mine = column < group * n;
  column = mine ? column : group * n - 1;
  const int r = column % n, head = key_head * group + column / n;
  const int visible = len + r + 1;
  const size_t row = (static_cast<size_t>(first + r) * c.n_heads + head) * 64;
  float4 qv[4];
#pragma unroll
  for (int i = 0; i < 4; i++) qv[i] = reinterpret_cast<const float4 *>(a.q + row + 16 * g)[i];

  Pages64 next = find(begin);
  Stage stage[2];
  load(next, stage[0]);
  next = find(begin + 64);

  // The query as bytes: the columns of the first product.
  v4i digit[3];
  float q_factor;
  {
    uint32_t big = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float x[4] = {qv[i].x, qv[i].y, qv[i].z, qv[i].w};
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const uint32_t bits = __float_as_uint(x[j]) & 0x7fffffffu;
        big = bits > big ? bits : big;
      }
    }
    auto p = __builtin_amdgcn_permlane16_swap(big, big, false, false);
    big = p[0] > p[1] ? p[0] : p[1];
    p = __builtin_amdgcn_permlane32_swap(big, big, false, false);
    big = p[0] > p[1] ? p[0] : p[1];
    const bool finite = big < 0x7f800000u;
    int e = !finite || big == 0 ? 0 : __builtin_amdgcn_frexp_expf(__uint_as_float(big));
    e = e < -96 ? -96 : e;
    // log2(e) / 8: scores in powers of two.
    q_factor = finite ? __builtin_ldexpf(0.180336880111120426f, e - 22) : __builtin_nanf("");
    // 1.5 2^23 + i holds the integer i in its low bits; adding 128 to each byte of
    // i and inverting their top bits leaves signed bytes whose weighted sum is i.
    auto bytes = [&](float f) {
      const float t = __builtin_ldexpf(f, 22 - e) + 12582912.0f;
      return (__float_as_uint(t) + (0x00808080u - 0x4b400000u)) ^ 0x00808080u;
    };
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint32_t w0 = bytes(qv[i].x), w1 = bytes(qv[i].y), w2 = bytes(qv[i].z), w3 = bytes(qv[i].w);
      const uint32_t a01 = __builtin_amdgcn_perm(w1, w0, 0x05010400u), a23 = __builtin_amdgcn_perm(w3, w2, 0x05010400u);
      const uint32_t b01 = __builtin_amdgcn_perm(w1, w0, 0x0c0c0602u), b23 = __builtin_amdgcn_perm(w3, w2, 0x0c0c0602u);
      digit[0][i] = static_cast<int>(__builtin_amdgcn_perm(a23, a01, 0x05040100u));
      digit[1][i] = static_cast<int>(__builtin_amdgcn_perm(a23, a01, 0x07060302u));
      digit[2][i] = static_cast<int>(__builtin_amdgcn_perm(b23, b01, 0x05040100u));
    }
  }

  const float ninf = -__builtin_inff();
  float m = ninf, den = 0.0f;
  int power = -300;  // 2^power above every block scale of the values so far
  v4f acc[4];
#pragma unroll
  for (int d = 0; d < 4; d++) acc[d] = v4f{0.0f, 0.0f, 0.0f, 0.0f};

  auto consume = [&](const Stage &s, int key0, auto masked) {
    constexpr bool kMasked = decltype(masked)::value;
    float p[16];
    const float factor = q_factor * s.k_scale;
#pragma unroll
    for (int t = 0; t < 4; t++) {
      const v4i zero = {0, 0, 0, 0};
      const v4i c0 = __builtin_amdgcn_mfma_i32_16x16x64_i8(s.k[t], digit[0], zero, 0, 0, 0);
      const v4i c1 = __builtin_amdgcn_mfma_i32_16x16x64_i8(s.k[t], digit[1], zero, 0, 0, 0);
      const v4i c2 = __builtin_amdgcn_mfma_i32_16x16x64_i8(s.k[t], digit[2], zero, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float sum = fmaf_(static_cast<float>(c2[i]), 65536.0f, static_cast<float>((c1[i] << 8) + c0[i]));
        p[4 * t + i] = sum * factor;
        if (kMasked && key0 + 16 * g + 4 * t + i >= visible) p[4 * t + i] = ninf;
      }
    }
    float top = p[0];
#pragma unroll
    for (int i = 1; i < 16; i++) top = __builtin_fmaxf(top, p[i]);
    top = __builtin_fmaxf(m, across_max(top));
    const float from = top == ninf ? 0.0f : top;
    const float widest = across_max(s.v_scale);
    int above = widest > 0.0f ? __builtin_amdgcn_frexp_expf(widest) : -300;
    above = __builtin_amdgcn_readfirstlane(above > power ? above : power);
    if (__any(top > m) || above > power) {
      const float keep = __builtin_amdgcn_exp2f(m - from);
      den = den * keep;
      const float scaled = __builtin_ldexpf(keep, power - above);
#pragma unroll
      for (int d = 0; d < 4; d++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[d][i] = acc[d][i] * scaled;
      m = top;
      power = above;
    }
    const float weight = __builtin_ldexpf(s.v_scale, 15 - power);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; i++) {
      p[i] = __builtin_amdgcn_exp2f(p[i] - from);
      sum = sum + p[i];
      p[i] = p[i] * weight;
      // A masked position's block may hold NaN.
      if (kMasked && key0 + 16 * g + i >= visible) p[i] = 0.0f;
    }
    den = den + sum;
#pragma unroll
    for (int step = 0; step < 2; step++) {
      // hi cut off, lo rounded to nearest: both conversions of hi (into the
      // product and into lo) are this one instruction's result.
      v8h hi, lo;
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        const float x = p[8 * step + j], y = p[8 * step + j + 1];
        const v2h pair = __builtin_bit_cast(v2h, __builtin_amdgcn_cvt_pkrtz(x, y));
        hi[j] = pair[0];
        hi[j + 1] = pair[1];
        lo[j] = static_cast<_Float16>(x - static_cast<float>(pair[0]));
        lo[j + 1] = static_cast<_Float16>(y - static_cast<float>(pair[1]));
      }
#pragma unroll
      for (int d = 0; d < 4; d++) {
        v8h v;
#pragma unroll
        for (int w = 0; w < 2; w++) {
          const uint32_t word = s.v[d][2 * step + w];
          const v2h bias = {static_cast<_Float16>(1152.0f), static_cast<_Float16>(1152.0f)};
          const v2h even = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, word, 0x04010400u)) - bias;
          const v2h odd = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, word, 0x04030402u)) - bias;
          v[4 * w] = even[0];
          v[4 * w + 1] = even[1];
          v[4 * w + 2] = odd[0];
          v[4 * w + 3] = odd[1];
        }
        acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, hi, acc[d], 0, 0, 0);
        acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, lo, acc[d], 0, 0, 0);
      }
    }
  };
  // While one 64 keys are worked on, the next are on their way, and the pages of
  // those after them.
  auto turn = [&](const Stage &now, Stage &then, int key0) {
    if (key0 + 64 < end) {
      load(next, then);
      next = find(key0 + 128);
    }
    if (key0 + 64 <= len)
      consume(now, key0, std::false_type());
    else
      consume(now, key0, std::true_type());
  };
  for (int key0 = begin; key0 < end; key0 += 128) {
    turn(stage[0], stage[1], key0);
    if (key0 + 64 < end) turn(stage[1], stage[0], key0 + 64);
  }

  den = across_sum(den);
  if (__any(missing) && lane == 0) c.refused[seq] = 1;
  // The four waves' states meet in LDS; thread: column tid / 16, dims 4 (tid % 16) .. + 3.
  __shared__ float s_m[4][16], s_den[4][16];
  __shared__ __attribute__((aligned(16))) float s_o[4][16][68];
  const float back = __builtin_ldexpf(1.0f, power - 15);
#pragma unroll
  for (int d = 0; d < 4; d++) {
    v4f o;
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] = acc[d][i] * back;
    *reinterpret_cast<v4f *>(&s_o[wave][l16][16 * d + 4 * g]) = o;
  }
  if (g == 0) {
    s_m[wave][l16] = m;
    s_den[wave][l16] = den;
  }
  __syncthreads();
  const int col = threadIdx.x / 16, dim = threadIdx.x % 16 * 4;
  const int out_column = 16 * tile + col;
  if (out_column >= group * n) return;
  const float top = __builtin_fmaxf(__builtin_fmaxf(s_m[0][col], s_m[1][col]), __builtin_fmaxf(s_m[2][col], s_m[3][col]));
  float total = 0.0f;
  v4f o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int w = 0; w < 4; w++) {
    const float f = state_weight(s_m[w][col], s_den[w][col], top);
    total = fmaf_(s_den[w][col], f, total);
    const v4f x = *reinterpret_cast<const v4f *>(&s_o[w][col][dim]);
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

// The parts of one row and head. Workgroup (head, row, sequence): thread = part
// for the weights, then 4 waves, lane = element, 8 parts of a wave in flight.
__global__ __launch_bounds__(256) void merge_kernel(AttendArgs a) {
  const Cache &c = a.c;
  const int head = blockIdx.x, r = blockIdx.y, seq = blockIdx.z;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  __shared__ float s_f[kMaxParts], s_top[4], s_den[4], s_o[4][64];
  int len, first, n;
  bool bad;
  const bool live = attend_span(a, seq, len, first, n, bad);
  if (bad && r == 0 && wave == 0) refuse_rows(a, seq, head, 1);
  if (!live || r >= n) return;
  const int parts = (len + n - 1) / a.chunk + 1;
  const size_t row = static_cast<size_t>(first + r) * c.n_heads + head, at = row * a.parts;
  float2 md = make_float2(-__builtin_inff(), 0.0f);
  if (tid < parts) md = reinterpret_cast<const float2 *>(a.part_md)[at + tid];
  float top = decode::wave_max(md.x);
  if (lane == 0) s_top[wave] = top;
  __syncthreads();
  top = __builtin_fmaxf(__builtin_fmaxf(s_top[0], s_top[1]), __builtin_fmaxf(s_top[2], s_top[3]));
  const float f = state_weight(md.x, md.y, top);
  s_f[tid] = f;
  const float den = decode::wave_sum(md.y * f);
  if (lane == 0) s_den[wave] = den;
  __syncthreads();
  float o = 0.0f;
  for (int p = wave; p < parts; p += 32) {
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = a.part_o[(at + (p + 4 * i < parts ? p + 4 * i : p)) * 64 + lane];
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (p + 4 * i < parts) o = fmaf_(x[i], s_f[p + 4 * i], o);
  }
  s_o[wave][lane] = o;
  __syncthreads();
  if (wave > 0) return;
  const float total = (s_den[0] + s_den[1]) + (s_den[2] + s_den[3]);
  o = (s_o[0][lane] + s_o[1][lane]) + (s_o[2][lane] + s_o[3][lane]);
  a.out[row * 64 + lane] = __fdiv_rn(o, total) * sink_factor(a.sinks, head, top, total);
}

// ---- pages of a sequence ---------------------------------------------------------
constexpr int kMapped = 240;
struct MapArgs {
  int32_t *table, *tags;  // of the sequence
  int first, count, shift, heads;
  int32_t pages[kMapped];
};

// Writes table entries, and forgets the FP32 blocks that stood in those pages.
__global__ __launch_bounds__(256) void map_kernel(MapArgs a) {
  for (int i = threadIdx.x; i < a.count; i += 256) a.table[a.first + i] = a.pages[i];
  for (int i = threadIdx.x; i < 2 * a.heads; i += 256) {
    const int block = a.tags[i], at = block >> a.shift;
    if (block >= 0 && at >= a.first && at < a.first + a.count) a.tags[i] = -1;
  }
}

__global__ __launch_bounds__(256) void fill_kernel(int32_t *to, size_t count, int32_t value) {
  for (size_t i = blockIdx.x * static_cast<size_t>(256) + threadIdx.x; i < count; i += static_cast<size_t>(gridDim.x) * 256)
    to[i] = value;
}

void free_pages(Pages *kv) {
  void *buffers[] = {kv->k_codes, kv->v_codes, kv->k_scales, kv->v_scales, kv->table, kv->open, kv->tags, kv->refused};
  for (void *p : buffers)
    if (p) (void)hipFree(p);
}

Cache cache_of(const Pages *kv, size_t rows, const int32_t *row_start, const int32_t *lens, size_t n_seqs) {
  Cache c = {};
  c.k_codes = kv->k_codes;
  c.v_codes = kv->v_codes;
  c.k_scales = kv->k_scales;
  c.v_scales = kv->v_scales;
  c.table = kv->table;
  c.open = kv->open;
  c.tags = kv->tags;
  c.refused = kv->refused;
  c.shift = kv->shift;
  c.seq_pages = static_cast<int>(kv->seq_pages);
  c.n_pages = static_cast<int>(kv->n_pages);
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
  const std::string at = std::string(name) + ": ";
  FOCR_REQUIRE(ctx && kv, FOCR_E_ARG, at + "null argument");
  FOCR_REQUIRE(kv->device == ctx->device, FOCR_E_ARG, at + "the cache is on another device than the context");
  FOCR_REQUIRE(n_seqs <= kv->n_seqs, FOCR_E_SHAPE, at + "more sequences than the cache has");
  FOCR_REQUIRE(rows < (size_t(1) << 24), FOCR_E_SHAPE, at + "too many rows");
  FOCR_REQUIRE(row_start || rows == n_seqs, FOCR_E_SHAPE, at + "without row_start every sequence has one row");
  FOCR_REQUIRE(rows == 0 || n_seqs == 0 || lens, FOCR_E_ARG, at + "null lengths");
  return FOCR_OK;
}

int launch_append(Ctx *ctx, const AppendArgs &a, bool qkv) {
  const Cache &c = a.c;
  // Units: n rows touch at most (n + 14) / 16 + 1 blocks, three of which are one
  // unit, so at most n / 16 units, or one.
  const int units = c.row_start ? c.rows / kBlock + (c.rows < c.n_seqs ? c.rows : c.n_seqs) : c.n_seqs;
  const int heads = c.key_heads + c.kv_heads + (qkv ? c.n_heads : 0);
  FOCR_HIP_CHECK(hipSetDevice(ctx->device));
  const dim3 grid(static_cast<unsigned>(units), static_cast<unsigned>((heads + 3) / 4));
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
  a.most = row_start ? static_cast<int>(rows < 8 ? rows : 8) : 1;
  const size_t group = kv->n_heads / kv->key_heads;
  a.tiles = static_cast<int>((group * a.most + 15) / 16);
  // Parts of whole 256 keys: about 2,048 workgroups (8 for each compute unit) where
  // all sequences are as long as the longest may be.
  const size_t heads = n_seqs * kv->key_heads * a.tiles;
  const size_t want = heads >= 2048 ? 1 : 2048 / heads;
  const size_t chunk = std::max((max_len + want - 1) / want, (max_len + kMaxParts - 1) / kMaxParts);
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
  hipLaunchKernelGGL(attend_kernel, dim3(static_cast<unsigned>(grid)), dim3(256), 0, ctx->stream, a);
  FOCR_HIP_CHECK(hipGetLastError());
  if (a.parts > 1) {
    hipLaunchKernelGGL(merge_kernel, dim3(static_cast<unsigned>(kv->n_heads), static_cast<unsigned>(a.most),
                                          static_cast<unsigned>(n_seqs)), dim3(256), 0, ctx->stream, a);
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
