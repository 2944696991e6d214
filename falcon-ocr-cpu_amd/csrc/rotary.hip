// The factors of rotary positions with several axes (rotary.hpp) for a step's rows:
// what the row steps (qkv_rows.hip, kv_split.hip, kv_pages.hip) take as `rope`. No
// reference counterpart on the device: its rotary_factors (src/model/rope.rs:103-142)
// builds them on the host, from the same sums for the same layout.
#include "rotary.hpp"

namespace focr {
namespace {

struct FactorArgs {
  const float *positions, *frequencies;
  float4 *out;
  int rows, slots;  // slots: twos of pairs in a row, n_heads * 16
  int rows_each;    // rows of a workgroup
};

// A thread keeps its two pairs' frequencies and walks rows. Bound: the factors written and
// the 64-bit arithmetic, 27 of 40 instructions for a pair with three axes, 3 to 4 us each
// for 6,544 rows of 16 heads (26.9 MB), which take 8.3 us with the launch. One row: 2.0, the launch.
template <int AXES>
__global__ __launch_bounds__(256) void factors_kernel(FactorArgs a) {
  const int slot = blockIdx.y * 256 + threadIdx.x;
  if (slot >= a.slots) return;
  double f[AXES][2];
#pragma unroll
  for (int x = 0; x < AXES; x++) {
    const float2 v = reinterpret_cast<const float2 *>(a.frequencies)[static_cast<size_t>(x) * a.slots + slot];
    f[x][0] = v.x;
    f[x][1] = v.y;
  }
  const int row0 = blockIdx.x * a.rows_each, rest = a.rows - row0, rows = rest < a.rows_each ? rest : a.rows_each;
  // Four rows' positions at a time, so that only the first are waited for.
  for (int base = 0; base < rows; base += 4) {
    float p[4][AXES];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float *at = a.positions + static_cast<size_t>(row0 + (base + i < rows ? base + i : base)) * AXES;
#pragma unroll
      for (int x = 0; x < AXES; x++) p[i][x] = at[x];
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if (base + i >= rows) break;
      double angle[2];
#pragma unroll
      for (int x = 0; x < AXES; x++)
#pragma unroll
        for (int j = 0; j < 2; j++) angle[j] = x == 0 ? p[i][x] * f[x][j] : __builtin_fma(static_cast<double>(p[i][x]), f[x][j], angle[j]);
      const float2 u = cos_sin(angle[0]), v = cos_sin(angle[1]);
      a.out[static_cast<size_t>(row0 + base + i) * a.slots + slot] = make_float4(u.x, u.y, v.x, v.y);
    }
  }
}

}  // namespace
}  // namespace focr

using namespace focr;

extern "C" int focr_rotary_factors(focr_ctx *handle, const float *positions, size_t rows, size_t axes,
                                   const float *frequencies, size_t n_heads, size_t head_dim, float *out) {
  Ctx *ctx = reinterpret_cast<Ctx *>(handle);
  FOCR_REQUIRE(ctx, FOCR_E_ARG, "focr_rotary_factors: null context");
  FOCR_REQUIRE(head_dim == 64, FOCR_E_UNSUPPORTED, "focr_rotary_factors: head_dim 64");
  FOCR_REQUIRE(axes >= 1 && axes <= kMaxAxes && n_heads > 0 && n_heads <= 1024, FOCR_E_SHAPE,
               "focr_rotary_factors: 1 to 4 axes, 1 to 1024 heads");
  FOCR_REQUIRE(rows < (size_t(1) << 31), FOCR_E_SHAPE, "focr_rotary_factors: too many rows");
  if (rows == 0) return FOCR_OK;
  FOCR_REQUIRE(positions && frequencies && out, FOCR_E_ARG, "focr_rotary_factors: null buffer");
  FOCR_REQUIRE(reinterpret_cast<uintptr_t>(out) % 16 == 0 && reinterpret_cast<uintptr_t>(frequencies) % 8 == 0, FOCR_E_ARG,
               "focr_rotary_factors: factors stand on 16 bytes, frequencies on 8");
  FactorArgs a = {};
  a.positions = positions;
  a.frequencies = frequencies;
  a.out = reinterpret_cast<float4 *>(out);
  a.rows = static_cast<int>(rows);
  a.slots = static_cast<int>(n_heads * 16);
  a.rows_each = static_cast<int>((rows + 2047) / 2048);
  const dim3 grid(static_cast<unsigned>((rows + a.rows_each - 1) / a.rows_each), static_cast<unsigned>((a.slots + 255) / 256));
  FOCR_HIP_CHECK(hipSetDevice(ctx->device));
  switch (axes) {
    case 1: hipLaunchKernelGGL(factors_kernel<1>, grid, dim3(256), 0, ctx->stream, a); break;
    case 2: hipLaunchKernelGGL(factors_kernel<2>, grid, dim3(256), 0, ctx->stream, a); break;
    case 3: hipLaunchKernelGGL(factors_kernel<3>, grid, dim3(256), 0, ctx->stream, a); break;
    default: hipLaunchKernelGGL(factors_kernel<4>, grid, dim3(256), 0, ctx->stream, a); break;
  }
  FOCR_HIP_CHECK(hipGetLastError());
  return FOCR_OK;
}
