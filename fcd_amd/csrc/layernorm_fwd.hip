// y = drop(act((x - mean) * rstd * gamma + beta)) (+ residual), the norm over a row: forward.
#include "fcd_layernorm.h"

namespace {

// The row in registers: mean, then the squares around it (two sums: one pass over E[x^2] - mean^2 would lose the spread of
// rows far from zero), then the result.  A workgroup walks over rows with its columns' parameters in registers and the next
// row's loads in flight.
template <typename T, int G, int NV, bool EPI>
__global__ __launch_bounds__(G > 64 ? G : 256) void ln_fwd_rows(LnArgs p) {
  constexpr int TH = G > 64 ? G : 256, RPB = TH / G, WAVES = RowSums<G, 1>::WAVES;
  __shared__ float sm[2 * WAVES];
  int turn = 0;
  if (EPI) drop_state(p.drop);
  const int lane = threadIdx.x % G, cols = (int)p.cols;
  const float fcols = (float)cols;
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
    const float mean = s[0] / fcols;
    s[0] = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int n = cols - (lane + k * G) * 8;
      float q = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[k][j] = j < n ? v[k][j] - mean : 0.f;
        q = fmaf(v[k][j], v[k][j], q);
      }
      s[0] += q;
    }
    RowSums<G, 1>::run(s, sm, turn);
    const float rstd = 1.f / sqrtf(s[0] / fcols + p.eps);
    if (lane == 0 && here && p.mean) {
      p.mean[row] = mean;
      p.rstd[row] = rstd;
    }
    T* out = (T*)p.out + row * p.ld_out;
#pragma unroll
    for (int k = 0; k < NV; ++k) arrive<T>(nx[k]);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (lane + k * G) * 8, n = here ? cols - c : 0;
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
      store8(out + c, n, u);
    }
  }
}

// Rows too long for registers: one workgroup per row, the row read again from cache for every pass.
template <typename T>
__global__ __launch_bounds__(1024) void ln_fwd_long(LnArgs p) {
  constexpr int TH = 1024;
  __shared__ float sm[2 * TH / 64];
  int turn = 0;
  drop_state(p.drop);
  for (long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* x = (const T*)p.x + row * p.ld_x;
    float s[1] = {0.f};
    for (long c = threadIdx.x * 8; c < p.cols; c += TH * 8) {
      float v[8];
      load8(x + c, p.cols - c, v);
      s[0] += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
    }
    RowSums<TH, 1>::run(s, sm, turn);
    const float mean = s[0] / (float)p.cols;
    s[0] = 0.f;
    for (long c = threadIdx.x * 8; c < p.cols; c += TH * 8) {
      const long n = p.cols - c;
      float v[8], q = 0.f;
      load8(x + c, n, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float d = j < n ? v[j] - mean : 0.f;
        q = fmaf(d, d, q);
      }
      s[0] += q;
    }
    RowSums<TH, 1>::run(s, sm, turn);
    const float rstd = 1.f / sqrtf(s[0] / (float)p.cols + p.eps);
    if (threadIdx.x == 0 && p.mean) {
      p.mean[row] = mean;
      p.rstd[row] = rstd;
    }
    for (long c = threadIdx.x * 8; c < p.cols; c += TH * 8) {
      const long n = p.cols - c;
      float v[8], u[8], ga[8], be[8];
      load8(x + c, n, v);
      load_param<T>(p.gamma, p.param_f32, c, n, 1.f, ga);
      load_param<T>(p.beta, p.param_f32, c, n, 0.f, be);
#pragma unroll
      for (int j = 0; j < 8; ++j) u[j] = fmaf((v[j] - mean) * rstd, ga[j], be[j]);
      ln_act8(u, p.act, v, nullptr, nullptr);
      if (p.drop.t) {
        uint32_t w[4];
        drop_draw8(p.drop, (uint64_t)(row * p.cols + c), w);
        drop_apply(p.drop, w, v);
      }
      if (p.res) {
        float r[8];
        load8((const T*)p.res + row * p.ld_res + c, n, r);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += r[j];
      }
      store8((T*)p.out + row * p.ld_out + c, n, v);
    }
  }
}

template <typename T>
void launch(const LnArgs& a, hipStream_t st) {
  const int64_t units = (a.cols + 7) / 8;
  const bool epi = a.act != 1.f || a.drop.t || a.res;
#define SHAPE(G, NV)                                                        \
  if (units <= G * NV) {                                                    \
    const int th = G > 64 ? G : 256;                                        \
    const long need = (a.rows + th / G - 1) / (th / G), full = 256 * (2048 / th); \
    const unsigned grid = (unsigned)(need < full ? need : full);            \
    if (epi) ln_fwd_rows<T, G, NV, true><<<grid, th, 0, st>>>(a);           \
    else ln_fwd_rows<T, G, NV, false><<<grid, th, 0, st>>>(a);              \
    return;                                                                 \
  }
  LN_FWD_SHAPES(SHAPE)
#undef SHAPE
  ln_fwd_long<T><<<(unsigned)(a.rows < 65536 ? a.rows : 65536), 1024, 0, st>>>(a);
}

}  // namespace

extern "C" int fcd_layernorm_fwd(const FcdLayerNormDesc* d, const void* x, const void* gamma, const void* beta,
                                 const void* residual, void* y, float* mean, float* rstd, void* stream) {
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
  if (d->rows == 0) return FCD_OK;
  a.x = x, a.gamma = gamma, a.beta = beta, a.res = residual, a.out = y, a.mean = mean, a.rstd = rstd;
  hipStream_t st = fcd_stream(stream);
  if (d->dtype == FCD_DT_F32) launch<float>(a, st);
  else if (d->dtype == FCD_DT_BF16) launch<bf16_t>(a, st);
  else launch<f16_t>(a, st);
  return fcd_check_launch(who);
}
