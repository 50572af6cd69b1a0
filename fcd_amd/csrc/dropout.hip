// Dropout from a counter-based generator: the mask is a function of (seed, offset, element index), so the backward pass
// computes it again instead of reading it.  One kernel serves both directions.
#include "fcd_rows.h"

namespace {

// 8 elements a thread and turn: x and the residual in, y out, one generator block between.  The units of a row start at the
// generator's blocks, not at the row's first element (memory takes any alignment; half a block would cost a whole one), so
// that a row's first unit may begin late and its last end early.  256 threads a row (WIDE), or 2^lt of them and several rows
// a workgroup; a tensor without gaps is one long row.
// Bound by memory, 16384 x 8192 bf16 95 us (5.7 TB/s), with a residual 134 (6.0, as without dropout: the best that a stream
// reads and writes here), at 17 vector instructions an element.  Rows that start anywhere in a block, 16384 x 8191 in rows of
// 8192: 132, of which 125 without dropout, for unaligned units and rows' ends (150 with units that start at the row and draw two
// blocks each).  65536 x 64 fp32 in rows of 68: 8 (35 with a workgroup per row).
template <typename T, bool WIDE>
__global__ __launch_bounds__(256) void dropout_kernel(const T* x, const T* res, T* y, long rows, long cols, long ld_x,
                                                      long ld_res, long ld_y, int lt, Drop d) {
  drop_state(d);
  if (WIDE) lt = 8;
  const int per_row = 1 << lt, rpb = 256 >> lt;
  for (long row = (long)blockIdx.y * rpb + (WIDE ? 0 : threadIdx.x >> lt); row < rows; row += (long)gridDim.y * rpb) {
    const T *xr = x + row * ld_x, *rr = res + row * ld_res;
    T* yr = y + row * ld_y;
    const int phase = (int)((row * cols) & 7);
    const uint64_t first = (uint64_t)(row * cols - phase);
    for (long u = ((long)blockIdx.x * per_row + (threadIdx.x & (per_row - 1))) * 8; u < cols + phase;
         u += (long)gridDim.x * per_row * 8) {
      const long c = u - phase;
      uint32_t w[4];
      if (c >= 0 && c + 8 <= cols) {
        typedef typename Oct<T>::type O;
        const O ox = *reinterpret_cast<const O*>(xr + c);
        O orr = {};
        if (res) orr = *reinterpret_cast<const O*>(rr + c);
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (float)ox[j];
        if (d.t) {
          drop_block(d, d.offset + ((first + u) >> 3), w);
          drop_apply(d, w, v);
        }
        O o;
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = (T)(res ? v[j] + (float)orr[j] : v[j]);
        *reinterpret_cast<O*>(yr + c) = o;
      } else {
        if (d.t) drop_block(d, d.offset + ((first + u) >> 3), w);
        for (int j = 0; j < 8; ++j) {
          if (c + j < 0 || c + j >= cols) continue;
          float v = (float)xr[c + j];
          if (d.t) {
            const uint32_t h = j < 2 ? w[0] : j < 4 ? w[1] : j < 6 ? w[2] : w[3];
            v = (j & 1 ? h : h << 16) > d.below ? v * d.scale : 0.f;
          }
          if (res) v += (float)rr[c + j];
          yr[c + j] = (T)v;
        }
      }
    }
  }
}

__global__ void dropout_take_kernel(uint64_t* state, uint64_t* taken, uint64_t blocks) {
  // (an atomic: calls on two streams at once take two ranges)
  taken[0] = state[0];
  taken[1] = atomicAdd((unsigned long long*)state + 1, (unsigned long long)blocks);
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
  FCD_TRY(fcd_check_apart(who, Bytes{"rng", rng, 16}, vy, rows, cols, es));
  if (rows == 0 || cols == 0) return FCD_OK;
  // a tensor without gaps is one long row: no division by the row length, no short ends
  if (rows > 1 && ld_x == cols && ld_y == cols && (!residual || ld_res == cols)) {
    cols *= rows;
    rows = 1;
  }
  int lt = 0;
  while (lt < 8 && ((int64_t)8 << lt) < cols + 7) ++lt;
  const int64_t bx = lt < 8 ? 1 : (cols + 7 + 2047) / 2048, by = (rows + (256 >> lt) - 1) / (256 >> lt);
  const dim3 grid((unsigned)(bx < (1 << 20) ? bx : (1 << 20)), (unsigned)(by < 32768 ? by : 32768));
  hipStream_t st = fcd_stream(stream);
#define LAUNCH(T)                                                                                                            \
  if (lt == 8)                                                                                                                \
    dropout_kernel<T, true><<<grid, 256, 0, st>>>((const T*)x, (const T*)residual, (T*)y, rows, cols, ld_x, ld_res, ld_y, lt, d); \
  else                                                                                                                        \
    dropout_kernel<T, false><<<grid, 256, 0, st>>>((const T*)x, (const T*)residual, (T*)y, rows, cols, ld_x, ld_res, ld_y, lt, d)
  if (dtype == FCD_DT_F32) {
    LAUNCH(float);
  } else if (dtype == FCD_DT_BF16) {
    LAUNCH(bf16_t);
  } else {
    LAUNCH(f16_t);
  }
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
