// Dropout from a counter-based generator: the mask is a function of (seed, offset, element index), so the backward pass
// computes it again instead of reading it.  One kernel serves both directions.
#include "fcd_rows.h"

namespace {

// 8 elements a thread and turn: x and the residual in, y out, one generator block between.  A workgroup stays in one row
// (blockIdx.y and further rows below it); a tensor without gaps is one long row.
template <typename T>
__global__ __launch_bounds__(256) void dropout_kernel(const T* x, const T* res, T* y, long rows, long cols, long ld_x,
                                                      long ld_res, long ld_y, Drop d) {
  drop_state(d);
  for (long row = blockIdx.y; row < rows; row += gridDim.y) {
    const T *xr = x + row * ld_x, *rr = res + row * ld_res;
    T* yr = y + row * ld_y;
    for (long c = ((long)blockIdx.x * 256 + threadIdx.x) * 8; c < cols; c += (long)gridDim.x * 256 * 8) {
      const long n = cols - c;
      float v[8], r[8];
      load8(xr + c, n, v);
      if (res) load8(rr + c, n, r);
      if (d.t) {
        uint32_t w[4];
        drop_draw8(d, (uint64_t)(row * cols + c), w);
        drop_apply(d, w, v);
      }
      if (res) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += r[j];
      }
      store8(yr + c, n, v);
    }
  }
}

__global__ void dropout_take_kernel(uint64_t* state, uint64_t* taken, uint64_t blocks) {
  const uint64_t seed = state[0], offset = state[1];
  taken[0] = seed;
  taken[1] = offset;
  state[1] = offset + blocks;
}

}  // namespace

extern "C" int fcd_dropout(const void* x, const void* residual, void* y, int64_t rows, int64_t cols, int64_t ld_x,
                           int64_t ld_res, int64_t ld_y, int dtype, double drop_p, uint64_t seed, uint64_t offset,
                           const uint64_t* rng, void* stream) {
  const char* who = "fcd_dropout";
  const int es = fcd_dt_bytes(dtype);
  FCD_REQUIRE(es, "%s: unknown element type %d", who, dtype);
  FCD_REQUIRE(rows >= 0 && cols >= 0, "%s: negative size", who);
  Drop d;
  FCD_TRY(fcd_make_drop(who, drop_p, seed, offset, rng, &d));
  const RowView vx{"x", x, ld_x}, vr{"residual", residual, ld_res}, vy{"y", y, ld_y};
  FCD_TRY(fcd_check_rows(who, vx, rows, cols, es, false));
  FCD_TRY(fcd_check_rows(who, vy, rows, cols, es, true));
  if (residual) FCD_TRY(fcd_check_rows(who, vr, rows, cols, es, false));
  FCD_TRY(fcd_check_apart(who, vy, vx, rows, cols, es, true));
  FCD_TRY(fcd_check_apart(who, vy, vr, rows, cols, es, true));
  if (rows == 0 || cols == 0) return FCD_OK;
  // a tensor without gaps is one long row: no division by the row length, no short ends
  if (rows > 1 && ld_x == cols && ld_y == cols && (!residual || ld_res == cols)) {
    cols *= rows;
    rows = 1;
  }
  const int64_t bx = (cols + 2047) / 2048;
  const dim3 grid((unsigned)(bx < (1 << 20) ? bx : (1 << 20)), (unsigned)(rows < 32768 ? rows : 32768));
  hipStream_t st = fcd_stream(stream);
#define LAUNCH(T)                                                                                                     \
  dropout_kernel<T><<<grid, 256, 0, st>>>((const T*)x, (const T*)residual, (T*)y, rows, cols, ld_x, ld_res, ld_y, d)
  if (dtype == FCD_DT_F32) LAUNCH(float);
  else if (dtype == FCD_DT_BF16) LAUNCH(bf16_t);
  else LAUNCH(f16_t);
#undef LAUNCH
  return fcd_check_launch(who);
}

extern "C" int fcd_dropout_take(uint64_t* state, uint64_t* taken, uint64_t blocks, void* stream) {
  const char* who = "fcd_dropout_take";
  FCD_REQUIRE(state && taken, "%s: NULL pointer", who);
  FCD_REQUIRE((((uintptr_t)state | (uintptr_t)taken) & 7u) == 0, "%s: the words must be 8-byte aligned", who);
  FCD_REQUIRE(taken + 2 <= state || state + 2 <= taken, "%s: taken overlaps state", who);
  dropout_take_kernel<<<1, 1, 0, fcd_stream(stream)>>>(state, taken, blocks);
  return fcd_check_launch(who);
}
