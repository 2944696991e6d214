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
constexpr int kPiece = 8192;  // tokens

struct SelectArgs {
  const float *logits;
  float *adjusted;
  int32_t *tokens;
  int32_t *history, *lengths;
  const float *penalties, *bias;
  const int32_t *bias_tokens;
  const uint32_t *allowed;
  ArgmaxPart *parts;
  uint32_t *arrived;
  int rows, vocab, cap, recent, n_bias, penalty_step, bias_step, words;
  size_t allowed_step;
  int segments, quads_each;  // workgroups of a row, and the fours of tokens of one
  int piece;                 // fours of tokens that LDS holds (0: no rule needs it)
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

// Workgroup: a row's fours of tokens from 4 * quads_each * segment on. Fours start where
// memory has 16-byte lines, so the first and the last of a row may be cut.
__global__ __launch_bounds__(256) void select_kernel(SelectArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint32_t words[];
  const int tid = threadIdx.x;
  const int row = blockIdx.x / a.segments, segment = blockIdx.x % a.segments;
  const float *const logits = a.logits + static_cast<size_t>(row) * a.vocab;
  float *const adjusted = a.adjusted ? a.adjusted + static_cast<size_t>(row) * a.vocab : nullptr;
  const int cut = reinterpret_cast<uintptr_t>(logits) / 4 % 4, all_quads = (a.vocab + cut + 3) / 4;
  const int begin = segment * a.quads_each, end = begin + a.quads_each < all_quads ? begin + a.quads_each : all_quads;
  const uint32_t *const allowed = a.allowed ? a.allowed + a.allowed_step * row : nullptr;
  const float *const penalty = a.penalties + static_cast<size_t>(a.penalty_step) * row;
  const float repetition = a.scan ? penalty[0] : 1.0f, presence = a.scan ? penalty[1] : 0.0f,
              frequency = a.scan ? penalty[2] : 0.0f;
  int length = a.lengths ? a.lengths[row] : 0;
  const int32_t *const history = a.history + static_cast<size_t>(row) * a.cap;
  const int counted = length < 0 ? 0 : length < a.cap ? length : a.cap;
  const int from = a.recent > 0 && counted > a.recent ? counted - a.recent : 0;
  const int32_t *const bias_tokens = a.bias_tokens + static_cast<size_t>(a.bias_step) * row;
  const float *const bias = a.bias + static_cast<size_t>(a.bias_step) * row;
  Best best = {-__builtin_inff(), -1, 0};
  const int step = a.piece > 0 ? a.piece : a.quads_each;
  for (int base = begin; base < end; base += step) {
    const int stop = base + step < end ? base + step : end;
    if (a.piece > 0) {
      for (int i = tid; i < stop - base; i += 256) reinterpret_cast<uint4 *>(words)[i] = make_uint4(0, 0, 0, 0);
      __syncthreads();
      const int first = 4 * base - cut;
      const uint32_t span = 4 * (stop - base);
      if (a.n_bias > 0) {
        // Of two biases for one token the later one counts.
        for (int i = tid; i < a.n_bias; i += 256) {
          const int token = bias_tokens[i];
          const uint32_t at = static_cast<uint32_t>(token - first);
          if (token >= 0 && token < a.vocab && at < span) atomicMax(words + at, static_cast<uint32_t>(i + 1) << kCountBits);
        }
        __syncthreads();
      }
      if (a.scan) {
        for (int i = from + tid; i < counted; i += 256) {
          const int token = history[i];
          const uint32_t at = static_cast<uint32_t>(token - first);
          if (token >= 0 && token < a.vocab && at < span) atomicAdd(words + at, 1u);
        }
        __syncthreads();
      }
    }
    for (int quad = base + tid; quad < stop; quad += 256) {
      const int token0 = 4 * quad - cut;
      const bool whole = token0 >= 0 && token0 + 4 <= a.vocab;
      float z[4];
      if (whole) {
        const float4 v = *reinterpret_cast<const float4 *>(logits + token0);
        z[0] = v.x;
        z[1] = v.y;
        z[2] = v.z;
        z[3] = v.w;
      } else {
#pragma unroll
        for (int j = 0; j < 4; j++) z[j] = token0 + j >= 0 && token0 + j < a.vocab ? logits[token0 + j] : -__builtin_inff();
      }
      if (a.piece > 0) {
        const uint4 w = reinterpret_cast<const uint4 *>(words)[quad - base];
        if (w.x | w.y | w.z | w.w) {
          const uint32_t rule[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const uint32_t count = rule[j] & kCountMask, number = rule[j] >> kCountBits;
            if (count > 0) {
              z[j] = z[j] > 0.0f ? __fdiv_rn(z[j], repetition) : z[j] * repetition;
              z[j] = z[j] - (static_cast<float>(count) * frequency + presence);
            }
            if (number > 0) z[j] = z[j] + bias[number - 1];
          }
        }
      }
      if (allowed) {
        const int word = token0 < 0 ? 0 : token0 >> 5;
        const uint32_t low = allowed[word], high = allowed[word + 1 < a.words ? word + 1 : word];
        const uint64_t both = static_cast<uint64_t>(high) << 32 | low;
        // The first four may begin before the row: their bits are those of its first tokens.
        const uint32_t bits = token0 < 0 ? low << -token0 : static_cast<uint32_t>(both >> (token0 & 31));
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (!(bits >> j & 1)) z[j] = -__builtin_inff();
      }
      if (adjusted) {
        if (whole && a.even) {
          *reinterpret_cast<float4 *>(adjusted + token0) = make_float4(z[0], z[1], z[2], z[3]);
        } else {
#pragma unroll
          for (int j = 0; j < 4; j++)
            if (token0 + j >= 0 && token0 + j < a.vocab) adjusted[token0 + j] = z[j];
        }
      }
#pragma unroll
      for (int j = 0; j < 4; j++) {
        if (z[j] > best.value) {
          best.value = z[j];
          best.index = token0 + j;
        }
        best.bad |= !(z[j] < __builtin_inff());
      }
    }
    if (a.piece > 0 && stop < end) __syncthreads();
  }
  if (!a.tokens) return;

  wave_best(best);
  __shared__ Best waves[4];
  if ((tid & 63) == 0) waves[tid >> 6] = best;
  __syncthreads();
  if (tid >= 64) return;
  best = waves[0];
#pragma unroll
  for (int w = 1; w < 4; w++) better(best, waves[w].value, waves[w].index, waves[w].bad);
  if (a.segments > 1) {
    // The row's last workgroup to arrive joins what all have found, in an order that
    // does not matter, and leaves the counter as it was.
    ArgmaxPart *const parts = a.parts + static_cast<size_t>(row) * a.segments;
    uint32_t before = 0;
    if (tid == 0) {
      parts[segment].value = best.value;
      parts[segment].index = best.index;
      parts[segment].nonfinite = best.bad;
      before = __hip_atomic_fetch_add(a.arrived + row, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
    }
    if (static_cast<int>(__builtin_amdgcn_readfirstlane(before)) != a.segments - 1) return;
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
    best = {-__builtin_inff(), -1, 0};
    for (int i = tid; i < a.segments; i += 64) better(best, parts[i].value, parts[i].index, parts[i].nonfinite);
    wave_best(best);
    if (tid == 0) a.arrived[row] = 0;
  }
  if (tid == 0) {
    const int token = best.bad ? -2 : best.index;
    a.tokens[row] = token;
    if (a.append && token >= 0 && length >= 0 && length < a.cap) {
      a.history[static_cast<size_t>(row) * a.cap + length] = token;
      a.lengths[row] = length + 1;
    }
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
  // A row is split while there are few rows, down to 1,024 tokens a workgroup.
  const size_t quads = (vocab + 6) / 4, want = rows <= Ctx::kSplitRows ? 1024 / rows : 1;
  const size_t segments = std::min(std::min<size_t>(want, Ctx::kSegments), (quads + 255) / 256);
  a.quads_each = static_cast<int>((quads + segments - 1) / segments);
  a.segments = static_cast<int>((quads + a.quads_each - 1) / a.quads_each);
  a.piece = a.scan || n_bias > 0 ? std::min(a.quads_each, kPiece / 4) : 0;
  FOCR_HIP_CHECK(hipSetDevice(ctx->device));
  if (a.segments > 1 && tokens) {
    const int rc = ensure_scratch(ctx, rows * a.segments * sizeof(ArgmaxPart));
    if (rc != FOCR_OK) return rc;
    a.parts = static_cast<ArgmaxPart *>(ctx->scratch);
    a.arrived = ctx->arrived;
  }
  hipLaunchKernelGGL(select_kernel, dim3(static_cast<unsigned>(rows * a.segments)), dim3(256), a.piece * 16, ctx->stream, a);
  FOCR_HIP_CHECK(hipGetLastError());
  return FOCR_OK;
}
