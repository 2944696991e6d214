// Rules on logits, and the greedy token. No reference counterpart: its greedy step takes
// the argmax of the logits as they are (src/runner/mod.rs:916-939).
//
// Row r has a history of tokens; c is how often token t stands among those counted.
//
//   z = logit;  c > 0: z = z > 0 ? z / repetition : z repetition,  z = z - (c frequency + presence)
//   a bias for t: z = z + bias;  t not allowed: z = -infinity
//
// every step rounded to FP32. The token is the lowest index of the largest z.
#include <algorithm>

#include "focr_internal.hpp"

namespace focr {
namespace {

// A word of LDS for each token of a piece: the count, and above it the number of the
// token's bias in the list (from 1 on; 0: none).
constexpr int kCountBits = 18;
constexpr uint32_t kCountMask = (1u << kCountBits) - 1;
constexpr int kThreads = 256;      // of a workgroup
constexpr int kPiece = 8192;       // tokens
static_assert(kPiece / 32 <= kThreads, "a mask word a thread");
constexpr int kHeldBiases = 1024;  // values in LDS

struct SelectArgs {
  const float *logits;
  float *adjusted;
  int32_t *tokens;
  int32_t *history, *lengths;
  const float *penalties, *bias;
  const int32_t *bias_tokens;
  const uint32_t *allowed;
  RowJoin *joins;
  int rows, vocab, cap, recent, n_bias, penalty_step, bias_step, words;
  size_t allowed_step;
  int segments, quads_each;  // workgroups of a row, and the fours of tokens of one
  int append, scan, even;    // scan: penalties are given; even: adjusted rows stand as logits' do
};

struct Best {
  float value;
  int index, bad;
};
__device__ __forceinline__ void better(Best &b, float value, int index, int bad) {
  if (index >= 0 && (b.index < 0 || value > b.value || (value == b.value && index < b.index))) {
    b.value = value;
    b.index = index;
  }
  b.bad |= bad;
}
__device__ __forceinline__ void wave_best(Best &b) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) {
    const float value = __shfl_xor(b.value, d);
    const int index = __shfl_xor(b.index, d), bad = __shfl_xor(b.bad, d);
    better(b, value, index, bad);
  }
}

// A list of tokens that a workgroup looks through: its first fours are loaded by begin, so
// that the trip to memory is not waited for there, the rest by each.
struct List {
  static constexpr int BATCH = 4;
  const int32_t *tokens;
  int from, to, head, fours;
  int4 front;
  int edge;

  // Fours that begin on 16 bytes, and up to three before and behind them (`edge`: thread
  // 0 .. 2 and 4 .. 6).
  __device__ __forceinline__ int edge_at() const {
    const int tid = threadIdx.x;
    if (tid < head - from) return from + tid;
    return tid >= 4 && tid - 4 < (to - head) % 4 ? head + 4 * fours + tid - 4 : -1;
  }
  __device__ __forceinline__ void begin(const int32_t *list, int first, int end) {
    tokens = list;
    from = first;
    to = end;
    head = from + static_cast<int>((16 - reinterpret_cast<uintptr_t>(tokens + from) % 16) / 4 % 4);
    head = head < to ? head : to;
    fours = (to - head) / 4;
    const int tid = threadIdx.x, at = edge_at();
    edge = at >= 0 ? tokens[at] : -1;
    if (tid < fours) front = reinterpret_cast<const int4 *>(tokens + head)[tid];
  }
  // add(place, number) for each token of the list that stands in first .. first + span - 1.
  template <typename Add>
  __device__ __forceinline__ void each(int first, int vocab, uint32_t span, const Add &add) {
    auto look = [&](int token, int i) {
      const uint32_t at = static_cast<uint32_t>(token - first);
      if (token >= 0 && token < vocab && at < span) add(at, i);
    };
    auto four = [&](const int4 &v, int number) {
      const int i = head + 4 * number;
      look(v.x, i);
      look(v.y, i + 1);
      look(v.z, i + 2);
      look(v.w, i + 3);
    };
    const int tid = threadIdx.x;
    look(edge, edge_at());
    if (tid < fours) four(front, tid);
    const int4 *const quads = reinterpret_cast<const int4 *>(tokens + head);
    for (int base = tid + kThreads; base < fours; base += BATCH * kThreads) {
      int4 v[BATCH];
#pragma unroll
      for (int j = 0; j < BATCH; j++) v[j] = quads[base + kThreads * j < fours ? base + kThreads * j : base];
#pragma unroll
      for (int j = 0; j < BATCH; j++)
        if (base + kThreads * j < fours) four(v[j], base + kThreads * j);
    }
  }
};

// Workgroup: a row's fours of tokens from quads_each * segment on, in pieces of up to
// kPiece tokens. All that a piece needs is asked for before anything is waited for: logits
// (in registers), mask, biases, history. Fours start where memory has 16-byte lines, so
// the first and the last of a row may be cut.
//
// Bound: the logits read, and written where they are kept. 256 rows of 131,072 with all
// rules and their logits kept take 72 us, 274 MB at 3.8 TB/s; 55 without rules (5.0, a copy's
// rate), 56 with the mask, 60 with penalties, 65 with 300 biases: every piece looks through
// the row's lists, and no logits are on their way meanwhile. 64 rows of 65,536 take 16 us,
// 8.0 without rules, 9.1 with the mask, 11.4 with 200 biases, 14.5 with penalties, of which
// 5 are the histories of up to 8,192 (eight fours a thread; with tokens spread evenly the
// same). One row 6.9 us, a launch, two trips to memory and three atomics one after another.
// Pieces of 4,096 tokens: 85 and 15.3; of 16,384 with 512 threads 69 and 14.7, one row and
// seven of 50,021 as they are.
template <bool RULES>
__global__ __launch_bounds__(kThreads) void select_kernel(SelectArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint32_t words[];
  constexpr int MOST = kPiece / 4 / kThreads;  // fours of a thread
  __shared__ uint32_t mask[kThreads + 2];
  __shared__ float held[RULES ? kHeldBiases : 1];
  const int tid = threadIdx.x;
  // Workgroups go to the 8 XCDs in turn: a row's share one, whose L2 has its history.
  const int turn = blockIdx.x / 8;
  const int row = a.rows < 8 ? blockIdx.x / a.segments : turn / a.segments * 8 + blockIdx.x % 8;
  const int segment = a.rows < 8 ? blockIdx.x % a.segments : turn % a.segments;
  if (row >= a.rows) return;
  const float *const logits = a.logits + static_cast<size_t>(row) * a.vocab;
  float *const adjusted = a.adjusted ? a.adjusted + static_cast<size_t>(row) * a.vocab : nullptr;
  const int cut = reinterpret_cast<uintptr_t>(logits) / 4 % 4, all_quads = (a.vocab + cut + 3) / 4;
  const int begin = segment * a.quads_each, end = begin + a.quads_each < all_quads ? begin + a.quads_each : all_quads;
  const int length = a.lengths ? a.lengths[row] : 0;
  float repetition = 1.0f, presence = 0.0f, frequency = 0.0f;
  if (RULES && a.scan) {
    const float *const penalty = a.penalties + static_cast<size_t>(a.penalty_step) * row;
    repetition = penalty[0];
    presence = penalty[1];
    frequency = penalty[2];
  }
  Best best = {-__builtin_inff(), -1, 0};
  for (int base = begin; base < end; base += kPiece / 4) {
    const int stop = base + kPiece / 4 < end ? base + kPiece / 4 : end, first = 4 * base - cut;
    float z[MOST][4];
#pragma unroll
    for (int i = 0; i < MOST; i++) {
      const int quad = base + tid + kThreads * i, token0 = 4 * quad - cut;
      if (quad < stop) {
        if (token0 >= 0 && token0 + 4 <= a.vocab) {
          const float4 v = *reinterpret_cast<const float4 *>(logits + token0);
          z[i][0] = v.x;
          z[i][1] = v.y;
          z[i][2] = v.z;
          z[i][3] = v.w;
        } else {
#pragma unroll
          for (int j = 0; j < 4; j++) z[i][j] = token0 + j >= 0 && token0 + j < a.vocab ? logits[token0 + j] : -__builtin_inff();
        }
      }
    }
    // The piece's mask from the word of its first token on.
    const int word0 = first < 0 ? 0 : first >> 5;
    uint32_t own_mask[2] = {0, 0};
    if (a.allowed) {
      const uint32_t *const allowed = a.allowed + a.allowed_step * row;
      if (word0 + tid < a.words) own_mask[0] = allowed[word0 + tid];
      if (tid < 2 && word0 + kThreads + tid < a.words) own_mask[1] = allowed[word0 + kThreads + tid];
    }
    List biases, history;
    if constexpr (RULES) {
      if (a.n_bias > 0) {
        biases.begin(a.bias_tokens + static_cast<size_t>(a.bias_step) * row, 0, a.n_bias);
        const float *const bias = a.bias + static_cast<size_t>(a.bias_step) * row;
        for (int i = tid; i < a.n_bias && i < kHeldBiases; i += kThreads) held[i] = bias[i];
      }
      if (a.scan) {
        const int counted = length < 0 ? 0 : length < a.cap ? length : a.cap;
        const int from = a.recent > 0 && counted > a.recent ? counted - a.recent : 0;
        history.begin(a.history + static_cast<size_t>(row) * a.cap, from, counted);
      }
      for (int i = tid; i < stop - base; i += kThreads) reinterpret_cast<uint4 *>(words)[i] = make_uint4(0, 0, 0, 0);
    }
    if (a.allowed) {
      mask[tid] = own_mask[0];
      if (tid < 2) mask[kThreads + tid] = own_mask[1];
    }
    __syncthreads();
    if constexpr (RULES) {
      const uint32_t span = 4 * (stop - base);
      if (a.n_bias > 0) {
        // Of two biases for one token the later one counts.
        biases.each(first, a.vocab, span, [&](uint32_t at, int i) { atomicMax(words + at, static_cast<uint32_t>(i + 1) << kCountBits); });
        __syncthreads();
      }
      if (a.scan) {
        history.each(first, a.vocab, span, [&](uint32_t at, int) { atomicAdd(words + at, 1u); });
        __syncthreads();
      }
    }
#pragma unroll
    for (int i = 0; i < MOST; i++) {
      const int quad = base + tid + kThreads * i, token0 = 4 * quad - cut;
      if (quad >= stop) continue;
      if constexpr (RULES) {
        const uint4 w = reinterpret_cast<const uint4 *>(words)[quad - base];
        if (w.x | w.y | w.z | w.w) {
          const uint32_t rule[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const uint32_t count = rule[j] & kCountMask, number = rule[j] >> kCountBits;
            if (count > 0) {
              z[i][j] = z[i][j] > 0.0f ? __fdiv_rn(z[i][j], repetition) : z[i][j] * repetition;
              z[i][j] = z[i][j] - (static_cast<float>(count) * frequency + presence);
            }
            if (number > 0)
              z[i][j] = z[i][j] + (number <= kHeldBiases ? held[number - 1] : a.bias[static_cast<size_t>(a.bias_step) * row + number - 1]);
          }
        }
      }
      if (a.allowed) {
        // Bits of four tokens, which two words may hold; what stands before the row has none.
        const int shift = token0 - 32 * word0, word = shift < 0 ? 0 : shift >> 5;
        const uint64_t both = static_cast<uint64_t>(mask[word + 1]) << 32 | mask[word];
        const uint32_t bits = shift < 0 ? static_cast<uint32_t>(both << -shift) : static_cast<uint32_t>(both >> (shift & 31));
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (!(bits >> j & 1)) z[i][j] = -__builtin_inff();
      }
      if (adjusted) {
        if (a.even && token0 >= 0 && token0 + 4 <= a.vocab) {
          *reinterpret_cast<float4 *>(adjusted + token0) = make_float4(z[i][0], z[i][1], z[i][2], z[i][3]);
        } else {
#pragma unroll
          for (int j = 0; j < 4; j++)
            if (token0 + j >= 0 && token0 + j < a.vocab) adjusted[token0 + j] = z[i][j];
        }
      }
#pragma unroll
      for (int j = 0; j < 4; j++) {
        if (z[i][j] > best.value) {
          best.value = z[i][j];
          best.index = token0 + j;
        }
        best.bad |= !(z[i][j] < __builtin_inff());
      }
    }
    if (stop < end) __syncthreads();
  }
  if (!a.tokens) return;

  wave_best(best);
  __shared__ Best waves[kThreads / 64];
  if ((tid & 63) == 0) waves[tid >> 6] = best;
  __syncthreads();
  if (tid > 0) return;
  best = waves[0];
#pragma unroll
  for (int w = 1; w < kThreads / 64; w++) better(best, waves[w].value, waves[w].index, waves[w].bad);
  int token = best.bad ? -2 : best.index;
  if (a.segments > 1) {
    // What the row's workgroups found is joined by the largest key: the value in the order
    // of its bits (both zeros alike), then the lower index; all ones for what is not
    // finite, 0 for nothing. The last to arrive reads it, and leaves key and counter at 0
    // for the next call. All of these are atomics on the device's memory, each waited for
    // before the next, so that no cache has to be written back.
    const uint32_t value = __float_as_uint(best.value + 0.0f);
    const uint64_t order = value >> 31 ? ~value : value | 0x80000000u;
    const unsigned long long key = best.bad ? ~uint64_t(0) : best.index < 0 ? 0 : order << 32 | (0xffffffffu - static_cast<uint32_t>(best.index));
    const unsigned long long held = __hip_atomic_fetch_max(&a.joins[row].key, key, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("s_waitcnt vmcnt(0)" ::"v"(held) : "memory");
    const uint32_t before = __hip_atomic_fetch_add(&a.joins[row].arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("s_waitcnt vmcnt(0)" ::"v"(before) : "memory");
    if (before != static_cast<uint32_t>(a.segments - 1)) return;
    const uint64_t most = __hip_atomic_exchange(&a.joins[row].key, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store(&a.joins[row].arrived, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    token = most == ~uint64_t(0) ? -2 : most == 0 ? -1 : static_cast<int>(0xffffffffu - static_cast<uint32_t>(most));
  }
  a.tokens[row] = token;
  if (a.append && token >= 0 && length >= 0 && length < a.cap) {
    a.history[static_cast<size_t>(row) * a.cap + length] = token;
    a.lengths[row] = length + 1;
  }
}

}  // namespace
}  // namespace focr

using namespace focr;

extern "C" int focr_logits_select(focr_ctx *handle, const float *logits, size_t rows, size_t vocab, int32_t *history,
                                  int32_t *lengths, size_t history_cap, size_t recent, const float *penalties,
                                  size_t penalty_rows, const int32_t *bias_tokens, const float *bias, size_t n_bias,
                                  size_t bias_rows, const uint32_t *allowed, size_t allowed_rows, int append,
                                  float *adjusted, int32_t *tokens) {
  Ctx *ctx = reinterpret_cast<Ctx *>(handle);
  FOCR_REQUIRE(ctx, FOCR_E_ARG, "focr_logits_select: null context");
  FOCR_REQUIRE(vocab > 0 && vocab < (size_t(1) << 30), FOCR_E_SHAPE, "focr_logits_select: 1 .. 2^30 - 1 tokens");
  FOCR_REQUIRE(rows < (size_t(1) << 24), FOCR_E_SHAPE, "focr_logits_select: too many rows");
  if (rows == 0) return FOCR_OK;
  FOCR_REQUIRE(logits && (adjusted || tokens), FOCR_E_ARG, "focr_logits_select: null buffer");
  FOCR_REQUIRE(reinterpret_cast<uintptr_t>(logits) % 4 == 0 && reinterpret_cast<uintptr_t>(adjusted) % 4 == 0, FOCR_E_ARG,
               "focr_logits_select: misaligned logits");
  const uintptr_t from = reinterpret_cast<uintptr_t>(logits), to = reinterpret_cast<uintptr_t>(adjusted), size = rows * vocab * 4;
  FOCR_REQUIRE(!adjusted || from == to || from + size <= to || to + size <= from, FOCR_E_ARG,
               "focr_logits_select: adjusted logits stand in the logits' place or in another");
  FOCR_REQUIRE(!history == !lengths, FOCR_E_ARG, "focr_logits_select: a history and its lengths");
  FOCR_REQUIRE(history || !(penalties || append), FOCR_E_ARG, "focr_logits_select: penalties and appending need a history");
  FOCR_REQUIRE(!append || tokens, FOCR_E_ARG, "focr_logits_select: appending needs the tokens");
  const size_t counted = recent > 0 && recent < history_cap ? recent : history_cap;
  FOCR_REQUIRE(!history || (history_cap > 0 && history_cap < (size_t(1) << 31)), FOCR_E_SHAPE, "focr_logits_select: history sizes");
  FOCR_REQUIRE(!penalties || counted <= kCountMask, FOCR_E_SHAPE, "focr_logits_select: penalties count at most 2^18 - 1 tokens");
  FOCR_REQUIRE(!penalties || penalty_rows == 1 || penalty_rows == rows, FOCR_E_SHAPE, "focr_logits_select: penalties of one row or of all");
  FOCR_REQUIRE(n_bias == 0 || (bias_tokens && bias), FOCR_E_ARG, "focr_logits_select: null biases");
  FOCR_REQUIRE(n_bias < (size_t(1) << (32 - kCountBits)), FOCR_E_SHAPE, "focr_logits_select: at most 2^14 - 1 biases");
  FOCR_REQUIRE(n_bias == 0 || bias_rows == 1 || bias_rows == rows, FOCR_E_SHAPE, "focr_logits_select: biases of one row or of all");
  FOCR_REQUIRE(!allowed || allowed_rows == 1 || allowed_rows == rows, FOCR_E_SHAPE, "focr_logits_select: masks of one row or of all");
  SelectArgs a = {};
  a.logits = logits;
  a.adjusted = adjusted;
  a.tokens = tokens;
  a.history = history;
  a.lengths = lengths;
  a.penalties = penalties;
  a.bias = bias;
  a.bias_tokens = bias_tokens;
  a.allowed = allowed;
  a.rows = static_cast<int>(rows);
  a.vocab = static_cast<int>(vocab);
  a.cap = static_cast<int>(history_cap);
  a.recent = static_cast<int>(recent < history_cap ? recent : 0);
  a.n_bias = static_cast<int>(n_bias);
  a.penalty_step = penalty_rows == 1 ? 0 : 3;
  a.bias_step = bias_rows == 1 ? 0 : static_cast<int>(n_bias);
  a.words = static_cast<int>((vocab + 31) / 32);
  a.allowed_step = allowed_rows == 1 ? 0 : a.words;
  a.append = append != 0;
  a.scan = penalties != nullptr;
  a.even = from % 16 == to % 16;
  // A workgroup for each piece of a row, and for a part of one, down to 1,024 tokens, while
  // there are few.
  const size_t quads = vocab % 4 == 0 ? (vocab + from % 16 / 4 + 3) / 4 : (vocab + 6) / 4, pieces = (quads + kPiece / 4 - 1) / (kPiece / 4);
  const size_t want = std::max(pieces, 512 / rows);
  const size_t segments = rows <= kJoinRows ? std::min(want, (quads + 255) / 256) : 1;
  a.quads_each = static_cast<int>((quads + segments - 1) / segments);
  a.segments = static_cast<int>((quads + a.quads_each - 1) / a.quads_each);
  const bool rules = a.scan || n_bias > 0;
  const size_t lds = rules ? std::min<size_t>(a.quads_each, kPiece / 4) * 16 : 0;
  const size_t grid = (rows < 8 ? rows : (rows + 7) / 8 * 8) * a.segments;
  FOCR_REQUIRE(grid < (size_t(1) << 31), FOCR_E_SHAPE, "focr_logits_select: too many rows and tokens");
  FOCR_HIP_CHECK(hipSetDevice(ctx->device));
  a.joins = ctx->joins;
  if (rules)
    hipLaunchKernelGGL(select_kernel<true>, dim3(static_cast<unsigned>(grid)), dim3(kThreads), lds, ctx->stream, a);
  else
    hipLaunchKernelGGL(select_kernel<false>, dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0, ctx->stream, a);
  FOCR_HIP_CHECK(hipGetLastError());
  return FOCR_OK;
}
