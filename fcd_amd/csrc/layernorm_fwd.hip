// y = drop(act((x - mean) * rstd * gamma + beta)) (+ residual), the norm over a row: forward.
#include "fcd_layernorm.h"

namespace {

// The row in registers: mean, then the squares around it (two sums: one pass over E[x^2] - mean^2 would lose the spread of
// rows far from zero), then the result.  A workgroup walks over rows with its columns' parameters in registers (fp32 gamma and
// beta are four times a bf16 row) and the next row's loads in flight; the grid is eight waves a SIMD (half of it: 65536 x 1024
// bf16 42.8 -> 44.7 us), or one workgroup of 1024, of which no second one fits (2048 x 12288 bf16 dropout with two 28.6, 26.4).
// Bound by memory: 16384 x 8192 bf16 95 us (5.6 TB/s; the best stream that reads and writes runs at 6.0), with dropout 97 to 116
// from process to process; 4096 x 4096 14, with SiLU and dropout 19.6; 8192 x 2048 with dropout 16.6; 65536 x 64 fp32 6.9, with
// leaky ReLU and dropout 7.8.  16384 x 8192 with dropout and a residual takes 23
// vector instructions an element, most of them the generator's.
template <typename T, int G, int NV, bool EPI>
__global__ __launch_bounds__(G > 64 ? G : 256) void ln_fwd_rows(LnArgs p) {
  constexpr int TH = G > 64 ? G : 256, RPB = TH / G, WAVES = RowSums<G, 1>::WAVES;
  __shared__ float sm[2 * WAVES];
  int turn = 0;
  if (EPI) drop_state(p.drop);
  const int lane = threadIdx.x % G, cols = (int)p.cols;
  const float fcols = (float)cols, inv = 1.f / fcols;
  float ga[NV][8], be[NV][8];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (lane + k * G) * 8;
    load_param<T>(p.gamma, p.param_f32, c, cols - c, 1.f, ga[k]);
    load_param<T>(p.beta, p.param_f32, c, cols - c, 0.f, be[k]);
  }
  typename Oct<T>::type nx[NV];
  auto fetch = [&](const void* t, long ld, long r, typename Oct<T>::type (&o)[NV]) {
    const T* x = (const T*)t + r * ld;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (lane + k * G) * 8;
      if (G >= 64 || r < p.rows) fetch8<T, G>(x, c, cols, o[k]);
    }
  };
  // G < 64: every thread of a wave makes the same number of turns, for the sums need whole groups; G >= 64: whole waves do
  long row = first_row<G, TH>();
  const long step = (long)gridDim.x * RPB;
  const long turns = (p.rows - (G >= 64 ? row : (long)blockIdx.x * RPB) + step - 1) / step;
  if (idle_wave<G>(cols)) {
    for (long it = 0; it < turns; ++it) {
      idle_sums<G, 1>(sm, turn);
      idle_sums<G, 1>(sm, turn);
    }
    return;
  }
  if (turns > 0) fetch(p.x, p.ld_x, row, nx);
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    arrive<T>(nx[k]);
  }
  for (long it = 0; it < turns; ++it, row += step) {
    const bool here = G >= 64 || row < p.rows;
    float v[NV][8];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      settle<T, G>(nx[k], cols, here ? cols - (lane + k * G) * 8 : 0);
      widen<T>(nx[k], v[k]);
    }
    typename Oct<T>::type rs[NV];
    if (EPI && p.res) fetch(p.res, p.ld_res, row, rs);
    if (it + 1 < turns) fetch(p.x, p.ld_x, row + step, nx);
    float s[1] = {0.f};
#pragma unroll
    for (int k = 0; k < NV; ++k)
      s[0] += ((v[k][0] + v[k][1]) + (v[k][2] + v[k][3])) + ((v[k][4] + v[k][5]) + (v[k][6] + v[k][7]));
    RowSums<G, 1>::run(s, sm, turn);
    // the quotient, corrected once by its remainder: exact where it is a number (rows without spread), and a tenth of a
    // division's instructions
    float mean = s[0] * inv;
    const float fine = fmaf(fmaf(-mean, fcols, s[0]), inv, mean);
    mean = fine == fine ? fine : mean;                       // (an infinite sum has no remainder)
    s[0] = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int n = cols - (lane + k * G) * 8;
      float q = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) v[k][j] -= mean;
      if (n < 8) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[k][j] = j < n ? v[k][j] : 0.f;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) q = fmaf(v[k][j], v[k][j], q);
      s[0] += q;
    }
    RowSums<G, 1>::run(s, sm, turn);
    // (the instruction takes a subnormal number, which eps = 0 lets through, for zero)
    const float var = fmaf(s[0], inv, p.eps);
    const bool tiny = var < 0x1p-126f;
    const float rstd = __builtin_amdgcn_rsqf(tiny ? var * 0x1p24f : var) * (tiny ? 0x1p12f : 1.f);
    if (lane == 0 && here && p.mean) {
      p.mean[row] = mean;
      p.rstd[row] = rstd;
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (lane + k * G) * 8, n = here ? cols - c : 0;
      if (k > 0 && G >= 64 && (__builtin_amdgcn_readfirstlane(lane & ~63) + k * G) * 8 >= cols) break;   // none in this wave
      float u[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) u[j] = fmaf(v[k][j] * rstd, ga[k][j], be[k][j]);
      if (EPI) {
        if (p.act != 1.f) {
          float a[8];
          ln_act8(u, p.act, a, nullptr, nullptr);
#pragma unroll
          for (int j = 0; j < 8; ++j) u[j] = a[j];
        }
        if (p.drop.t) {
          uint32_t w[4];
          drop_draw8(p.drop, (uint64_t)(row * cols + c), w);
          drop_apply(p.drop, w, u);
        }
        if (p.res) {
          float r[8];
          settle<T, G>(rs[k], cols, n);
          widen<T>(rs[k], r);
#pragma unroll
          for (int j = 0; j < 8; ++j) u[j] += r[j];
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) v[k][j] = u[j];
    }
    T* out = (T*)p.out + row * p.ld_out;
#pragma unroll
    for (int k = 0; k < NV; ++k) arrive<T>(nx[k]);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (lane + k * G) * 8;
      store8(out + c, here ? cols - c : 0, v[k]);
    }
  }
}

// Split rows, 1: mean and sum of squares around it of a chunk.
template <typename T>
__global__ __launch_bounds__(256) void ln_fwd_chunks(LnArgs p, long chunks) {
  __shared__ float sm[2 * 4];
  int turn = 0;
  for (long item = blockIdx.x; item < p.rows * chunks; item += gridDim.x) {
    const long row = item / chunks, c0 = (item - row * chunks) * CHUNK;
    const T* x = (const T*)p.x + row * p.ld_x;
    const float count = (float)(p.cols - c0 < CHUNK ? p.cols - c0 : CHUNK);
    float v[4][8], s[1] = {0.f};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const long c = c0 + (threadIdx.x + k * 256) * 8;
      load8(x + c, p.cols - c, v[k]);
      s[0] += ((v[k][0] + v[k][1]) + (v[k][2] + v[k][3])) + ((v[k][4] + v[k][5]) + (v[k][6] + v[k][7]));
    }
    RowSums<256, 1>::run(s, sm, turn);
    const float mean = s[0] / count;
    s[0] = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const long n = p.cols - c0 - (threadIdx.x + k * 256) * 8;
      float q = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float d = j < n ? v[k][j] - mean : 0.f;
        q = fmaf(d, d, q);
      }
      s[0] += q;
    }
    RowSums<256, 1>::run(s, sm, turn);
    if (threadIdx.x == 0) {
      p.chunk[item * 2] = mean;
      p.chunk[item * 2 + 1] = s[0];
    }
  }
}

// 2: the chunks of a row joined: sum of squares = those around the chunks' means + the means' own spread.
__global__ __launch_bounds__(256) void ln_fwd_join(LnArgs p, long chunks) {
  const int lane = threadIdx.x & 63;
  const float cols = (float)p.cols, last = (float)(p.cols - (chunks - 1) * CHUNK);
  for (long row = (long)blockIdx.x * 4 + (threadIdx.x >> 6); row < p.rows; row += (long)gridDim.x * 4) {
    const float* part = p.chunk + row * chunks * 2;
    float s = 0.f, q = 0.f;
    for (long i = lane; i < chunks; i += 64) s += part[i * 2] * (i + 1 < chunks ? (float)CHUNK : last);
    const float mean = lanes_sum<64>(s) / cols;
    for (long i = lane; i < chunks; i += 64) {
      const float d = part[i * 2] - mean;
      q += fmaf(d * d, i + 1 < chunks ? (float)CHUNK : last, part[i * 2 + 1]);
    }
    const float rstd = 1.f / sqrtf(lanes_sum<64>(q) / cols + p.eps);
    if (lane == 0) {
      p.row[row * 2] = mean;
      p.row[row * 2 + 1] = rstd;
      if (p.mean) {
        p.mean[row] = mean;
        p.rstd[row] = rstd;
      }
    }
  }
}

// 3: the result.
template <typename T>
__global__ __launch_bounds__(256) void ln_fwd_stream(LnArgs p) {
  drop_state(p.drop);
  const long c = ((long)blockIdx.x * 256 + threadIdx.x) * 8, n = p.cols - c;
  if (n <= 0) return;
  float ga[8], be[8];
  load_param<T>(p.gamma, p.param_f32, c, n, 1.f, ga);
  load_param<T>(p.beta, p.param_f32, c, n, 0.f, be);
  for (long row = blockIdx.y; row < p.rows; row += gridDim.y) {
    const float mean = p.row[row * 2], rstd = p.row[row * 2 + 1];
    float v[8], u[8], r[8];
    load8((const T*)p.x + row * p.ld_x + c, n, v);
    if (p.res) load8((const T*)p.res + row * p.ld_res + c, n, r);
#pragma unroll
    for (int j = 0; j < 8; ++j) u[j] = fmaf((v[j] - mean) * rstd, ga[j], be[j]);
    if (p.act != 1.f) {
      ln_act8(u, p.act, v, nullptr, nullptr);
#pragma unroll
      for (int j = 0; j < 8; ++j) u[j] = v[j];
    }
    if (p.drop.t) {
      uint32_t w[4];
      drop_draw8(p.drop, (uint64_t)(row * p.cols + c), w);
      drop_apply(p.drop, w, u);
    }
    if (p.res) {
#pragma unroll
      for (int j = 0; j < 8; ++j) u[j] += r[j];
    }
    store8((T*)p.out + row * p.ld_out + c, n, u);
  }
}

template <typename T>
void launch(const LnArgs& a, hipStream_t st) {
  const int64_t units = (a.cols + 7) / 8;
  const bool epi = a.act != 1.f || a.drop.t || a.res;
#define SHAPE(G, NV)                                                        \
  if (units <= G * NV) {                                                    \
    const int th = G > 64 ? G : 256;                                        \
    const long need = (a.rows + th / G - 1) / (th / G), full = 256 * (G == 1024 ? 1 : 2048 / th); \
    const unsigned grid = (unsigned)(need < full ? need : full);            \
    if (epi) ln_fwd_rows<T, G, NV, true><<<grid, th, 0, st>>>(a);           \
    else ln_fwd_rows<T, G, NV, false><<<grid, th, 0, st>>>(a);              \
    return;                                                                 \
  }
  LN_FWD_SHAPES(SHAPE)
#undef SHAPE
  const long chunks = ln_chunks(a.cols);
  ln_fwd_chunks<T><<<ln_items(a.rows, a.cols), 256, 0, st>>>(a, chunks);
  ln_fwd_join<<<ln_join_grid(a.rows), 256, 0, st>>>(a, chunks);
  ln_fwd_stream<T><<<ln_stream_grid(a.rows, a.cols), 256, 0, st>>>(a);
}

}  // namespace

extern "C" int fcd_layernorm_fwd(const FcdLayerNormDesc* d, const void* x, const void* gamma, const void* beta,
                                 const void* residual, void* y, float* mean, float* rstd, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  const char* who = "fcd_layernorm_fwd";
  LnArgs a;
  FCD_TRY(ln_check(who, d, &a));
  const int es = fcd_dt_bytes(d->dtype);
  const RowView vx{"x", x, d->ld_x}, vr{"residual", residual, d->ld_res}, vy{"y", y, d->ld_out};
  FCD_TRY(fcd_check_rows(who, vx, d->rows, d->cols, es, false));
  FCD_TRY(fcd_check_rows(who, vy, d->rows, d->cols, es, true));
  if (residual) FCD_TRY(fcd_check_rows(who, vr, d->rows, d->cols, es, false));
  FCD_TRY(fcd_check_apart(who, vy, vx, d->rows, d->cols, es, true));
  FCD_TRY(fcd_check_apart(who, vy, vr, d->rows, d->cols, es, true));
  FCD_TRY(ln_check_vectors(who, d, gamma, beta, mean, rstd));
  FCD_REQUIRE(!mean == !rstd, "%s: mean and rstd go together", who);
  FCD_TRY(ln_check_scratch(who, d, FCD_LN_FWD, nullptr, nullptr, workspace, workspace_bytes, &a));
  const int64_t ps = fcd_dt_bytes(d->param_dtype) * d->cols, ss = 4 * d->rows;
  const Bytes written[] = {{"mean", mean, ss}, {"rstd", rstd, ss}, {"workspace", workspace, (int64_t)workspace_bytes}};
  const Bytes read[] = {{"gamma", gamma, ps}, {"beta", beta, ps}, {"rng", d->rng, 16}};
  const RowView rows[] = {vx, vr, vy};
  FCD_TRY(ln_check_apart(who, d, written, 3, read, 3, rows, 3));
  for (const Bytes& b : read) FCD_TRY(fcd_check_apart(who, b, vy, d->rows, d->cols, es));
  if (d->rows == 0) return FCD_OK;
  a.x = x, a.gamma = gamma, a.beta = beta, a.res = residual, a.out = y, a.mean = mean, a.rstd = rstd;
  hipStream_t st = fcd_stream(stream);
  if (d->dtype == FCD_DT_F32) launch<float>(a, st);
  else if (d->dtype == FCD_DT_BF16) launch<bf16_t>(a, st);
  else launch<f16_t>(a, st);
  return fcd_check_launch(who);
}
