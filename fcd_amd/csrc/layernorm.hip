// Layer norm over the last axis with activation, dropout and residual fused; its backward with the affine gradients; the
// backward of that backward (gradient penalty).  fp32 sums, one rounding to the element type at the end.
#include "fcd_rows.h"

namespace {

struct LnArgs {
  const void *x, *res, *gy, *ggx, *gamma, *beta;
  void *out, *ggy;
  float *mean, *rstd;      // written by fwd, read by bwd / bwd2
  float* partial;          // [gridDim.x][2][cols]: this workgroup's sums of dgamma and dbeta; or NULL
  long rows, cols, ld_x, ld_res, ld_gy, ld_ggx, ld_out, ld_ggy;
  float eps, act;
  int param_f32;
  Drop drop;
};

template <typename T>
__device__ __forceinline__ void load_param(const void* p, int f32, long c, long n, float none, float (&v)[8]) {
  if (!p) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = none;
  } else if (f32) {
    load8((const float*)p + c, n, v);
  } else {
    load8((const T*)p + c, n, v);
  }
}

// Sums of K values over the workgroup, in every thread.
template <int TH, int K>
__device__ __forceinline__ void block_sums(float (&s)[K], float* sm) {
#pragma unroll
  for (int k = 0; k < K; ++k) s[k] = wave_sum(s[k]);
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  __syncthreads();
  if (lane == 0)
#pragma unroll
    for (int k = 0; k < K; ++k) sm[w * K + k] = s[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < TH / 64; ++i) t += sm[i * K + k];
    s[k] = t;
  }
}

// ---------------------------------------------------------------- any row length -------
// One workgroup per row, the row read again from cache for every pass.
template <typename T, int TH>
__global__ __launch_bounds__(TH) void ln_fwd_long(LnArgs p) {
  __shared__ float sm[TH / 64];
  drop_state(p.drop);
  for (long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* x = (const T*)p.x + row * p.ld_x;
    float s[1] = {0.f};
    for (long c = threadIdx.x * 8; c < p.cols; c += TH * 8) {
      float v[8];
      load8(x + c, p.cols - c, v);
#pragma unroll
      for (int j = 1; j < 8; ++j) v[0] += v[j];
      s[0] += v[0];
    }
    block_sums<TH>(s, sm);
    const float mean = s[0] / (float)p.cols;
    s[0] = 0.f;
    for (long c = threadIdx.x * 8; c < p.cols; c += TH * 8) {
      const long n = p.cols - c;
      float v[8];
      load8(x + c, n, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) s[0] += j < n ? (v[j] - mean) * (v[j] - mean) : 0.f;
    }
    block_sums<TH>(s, sm);
    const float rstd = 1.f / sqrtf(s[0] / (float)p.cols + p.eps);
    if (threadIdx.x == 0 && p.mean) {
      p.mean[row] = mean;
      p.rstd[row] = rstd;
    }
    for (long c = threadIdx.x * 8; c < p.cols; c += TH * 8) {
      const long n = p.cols - c;
      float v[8], ga[8], be[8];
      load8(x + c, n, v);
      load_param<T>(p.gamma, p.param_f32, c, n, 1.f, ga);
      load_param<T>(p.beta, p.param_f32, c, n, 0.f, be);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = act_value((v[j] - mean) * rstd * ga[j] + be[j], p.act);
      if (p.drop.t) drop_apply(p.drop, drop_keep8(p.drop, (uint64_t)(row * p.cols + c)), v);
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

// What the backward passes need of 8 elements: xhat, g1 = drop(gy) act'(u), a = g1 gamma; elements past the row's end: 0.
struct Eight {
  float xh[8], gy[8], u[8], ga[8], g1[8], a[8];
  uint32_t keep;
};

template <typename T>
__device__ __forceinline__ void load_eight(const LnArgs& p, long row, long c, float mean, float rstd, Eight& e) {
  const long n = p.cols - c;
  float be[8];
  load8((const T*)p.x + row * p.ld_x + c, n, e.xh);
  load8((const T*)p.gy + row * p.ld_gy + c, n, e.gy);
  load_param<T>(p.gamma, p.param_f32, c, n, 1.f, e.ga);
  load_param<T>(p.beta, p.param_f32, c, n, 0.f, be);
  e.keep = 0xff;
  if (p.drop.t) {
    e.keep = drop_keep8(p.drop, (uint64_t)(row * p.cols + c));
    drop_apply(p.drop, e.keep, e.gy);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    e.xh[j] = j < n ? (e.xh[j] - mean) * rstd : 0.f;
    e.u[j] = e.xh[j] * e.ga[j] + be[j];
    e.g1[j] = j < n ? e.gy[j] * act_slope_at(e.u[j], p.act) : 0.f;
    e.a[j] = e.g1[j] * e.ga[j];
  }
}

// Adds to this workgroup's sums; a thread meets the same columns in every row, so nothing else touches them.
__device__ __forceinline__ void add_partial(float* p, long n, bool first, const float (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < n) p[j] = first ? v[j] : p[j] + v[j];
}

template <typename T, int TH>
__global__ __launch_bounds__(TH) void ln_bwd_long(LnArgs p) {
  __shared__ float sm[TH / 64 * 2];
  drop_state(p.drop);
  const float inv = 1.f / (float)p.cols;
  for (long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const float mean = p.mean[row], rstd = p.rstd[row];
    float s[2] = {0.f, 0.f};
    for (long c = threadIdx.x * 8; c < p.cols; c += TH * 8) {
      Eight e;
      load_eight<T>(p, row, c, mean, rstd, e);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        s[0] += e.a[j];
        s[1] += e.a[j] * e.xh[j];
      }
    }
    block_sums<TH>(s, sm);
    const float am = s[0] * inv, ax = s[1] * inv;
    for (long c = threadIdx.x * 8; c < p.cols; c += TH * 8) {
      const long n = p.cols - c;
      Eight e;
      load_eight<T>(p, row, c, mean, rstd, e);
      float dx[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) dx[j] = rstd * (e.a[j] - am - e.xh[j] * ax);
      if (p.partial) {
        float* part = p.partial + (long)blockIdx.x * 2 * p.cols + c;
        float dg[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) dg[j] = e.g1[j] * e.xh[j];
        add_partial(part, n, row == blockIdx.x, dg);
        add_partial(part + p.cols, n, row == blockIdx.x, e.g1);
      }
      store8((T*)p.out + row * p.ld_out + c, n, dx);
    }
  }
}

template <typename T, int TH>
__global__ __launch_bounds__(TH) void ln_bwd2_long(LnArgs p) {
  __shared__ float sm[TH / 64 * 5];
  drop_state(p.drop);
  const float inv = 1.f / (float)p.cols;
  const bool smooth = p.act > 1.f;
  for (long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const float mean = p.mean[row], rstd = p.rstd[row];
    float s[5] = {0.f, 0.f, 0.f, 0.f, 0.f};
    for (long c = threadIdx.x * 8; c < p.cols; c += TH * 8) {
      Eight e;
      float v[8];
      load_eight<T>(p, row, c, mean, rstd, e);
      load8((const T*)p.ggx + row * p.ld_ggx + c, p.cols - c, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        s[0] += e.a[j];
        s[1] += e.a[j] * e.xh[j];
        s[2] += v[j];
        s[3] += v[j] * e.xh[j];
        s[4] += v[j] * e.a[j];
      }
    }
    block_sums<TH>(s, sm);
    const float am = s[0] * inv, ax = s[1] * inv, vm = s[2] * inv, vx = s[3] * inv;
    const float sv = s[4] * inv - vm * am - vx * ax;
    float q2[2] = {0.f, 0.f};
    if (smooth) {
      for (long c = threadIdx.x * 8; c < p.cols; c += TH * 8) {
        Eight e;
        float v[8];
        load_eight<T>(p, row, c, mean, rstd, e);
        load8((const T*)p.ggx + row * p.ld_ggx + c, p.cols - c, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float t = rstd * (v[j] - vm - e.xh[j] * vx);
          const float qg = j < p.cols - c ? e.gy[j] * act_curv_at(e.u[j], p.act) * e.ga[j] * t * e.ga[j] : 0.f;
          q2[0] += qg;
          q2[1] += qg * e.xh[j];
        }
      }
      block_sums<TH>(q2, sm);
    }
    const float hm = q2[0] * inv - rstd * (vm * ax + am * vx), hx = q2[1] * inv - 2.f * rstd * vx * ax;
    for (long c = threadIdx.x * 8; c < p.cols; c += TH * 8) {
      const long n = p.cols - c;
      Eight e;
      float v[8], gg[8], gx[8], dg[8], q[8];
      load_eight<T>(p, row, c, mean, rstd, e);
      load8((const T*)p.ggx + row * p.ld_ggx + c, n, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float t = rstd * (v[j] - vm - e.xh[j] * vx);
        q[j] = smooth ? e.gy[j] * act_curv_at(e.u[j], p.act) * e.ga[j] * t : 0.f;
        gg[j] = act_slope_at(e.u[j], p.act) * e.ga[j] * t;
        const float h = q[j] * e.ga[j] - rstd * (v[j] * ax + e.a[j] * vx);
        gx[j] = rstd * (h - hm - e.xh[j] * hx) - sv * rstd * rstd * e.xh[j];
        dg[j] = e.g1[j] * t + q[j] * e.xh[j];
      }
      if (p.drop.t) drop_apply(p.drop, e.keep, gg);
      if (p.partial) {
        float* part = p.partial + (long)blockIdx.x * 2 * p.cols + c;
        add_partial(part, n, row == blockIdx.x, dg);
        add_partial(part + p.cols, n, row == blockIdx.x, q);
      }
      store8((T*)p.ggy + row * p.ld_ggy + c, n, gg);
      store8((T*)p.out + row * p.ld_out + c, n, gx);
    }
  }
}

// dgamma (blockIdx.y 0) / dbeta (1): the workgroups' sums of one column, added in order.
template <typename P>
__global__ __launch_bounds__(256) void ln_affine_reduce(const float* partial, int groups, long cols, P* dgamma, P* dbeta,
                                                        int accumulate) {
  __shared__ float sm[4][64];
  P* out = blockIdx.y ? dbeta : dgamma;
  if (!out) return;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const long c = (long)blockIdx.x * 64 + lane;
  float s = 0.f;
  if (c < cols)
    for (int g = w; g < groups; g += 4) s += partial[((long)g * 2 + blockIdx.y) * cols + c];
  sm[w][lane] = s;
  __syncthreads();
  if (w == 0 && c < cols) {
    s = sm[0][lane] + sm[1][lane] + sm[2][lane] + sm[3][lane];
    out[c] = (P)(accumulate ? (float)out[c] + s : s);
  }
}

constexpr int LN_GROUPS = 256;   // workgroups that keep sums of their own

int64_t ln_groups(int64_t rows) { return rows < LN_GROUPS ? rows : LN_GROUPS; }

int ln_check(const char* who, const FcdLayerNormDesc* d, LnArgs* a) {
  FCD_REQUIRE(d, "%s: NULL descriptor", who);
  FCD_REQUIRE(fcd_dt_bytes(d->dtype), "%s: unknown element type %d", who, d->dtype);
  FCD_REQUIRE(d->param_dtype == FCD_DT_F32 || d->param_dtype == d->dtype, "%s: parameters must be fp32 or of x's type", who);
  FCD_REQUIRE(d->rows >= 0, "%s: negative number of rows", who);
  FCD_REQUIRE(d->cols >= 1 && d->cols < (int64_t)1 << 31, "%s: %lld columns (1 ... 2^31 - 1)", who, (long long)d->cols);
  FCD_REQUIRE(d->rows < (int64_t)1 << 58 && (__int128)d->rows * d->cols < (__int128)1 << 58, "%s: too many elements", who);
  FCD_REQUIRE(d->eps >= 0.f && d->eps <= 3.4e38f, "%s: eps must be finite and not negative", who);
  FCD_REQUIRE((d->act >= 0.f && d->act <= 1.f) || d->act == FCD_ACT_SILU || d->act == FCD_ACT_MISH,
              "%s: unknown activation code %g", who, (double)d->act);
  *a = LnArgs{};
  FCD_TRY(fcd_make_drop(who, d->drop_p, d->seed, d->offset, d->rng, &a->drop));
  a->rows = d->rows, a->cols = d->cols;
  a->ld_x = d->ld_x, a->ld_res = d->ld_res, a->ld_gy = d->ld_gy, a->ld_ggx = d->ld_ggx, a->ld_out = d->ld_out;
  a->ld_ggy = d->ld_ggy;
  a->eps = d->eps, a->act = d->act;
  a->param_f32 = d->param_dtype == FCD_DT_F32;
  return FCD_OK;
}

int ln_check_vectors(const char* who, const FcdLayerNormDesc* d, const void* gamma, const void* beta, const void* mean,
                     const void* rstd) {
  const uintptr_t m = (uintptr_t)(fcd_dt_bytes(d->param_dtype) - 1);
  FCD_REQUIRE((((uintptr_t)gamma | (uintptr_t)beta) & m) == 0, "%s: gamma / beta are not aligned to their element type", who);
  FCD_REQUIRE((((uintptr_t)mean | (uintptr_t)rstd) & 3u) == 0, "%s: mean / rstd are not 4-byte aligned", who);
  return FCD_OK;
}

template <typename P>
int ln_finish(const char* who, const LnArgs& a, int groups, void* dgamma, void* dbeta, int accumulate, hipStream_t st) {
  ln_affine_reduce<P><<<dim3((unsigned)((a.cols + 63) / 64), 2), 256, 0, st>>>(a.partial, groups, a.cols, (P*)dgamma, (P*)dbeta,
                                                                               accumulate);
  return fcd_check_launch(who);
}

int ln_finish(const char* who, const FcdLayerNormDesc* d, const LnArgs& a, int groups, void* dgamma, void* dbeta, int accumulate,
              hipStream_t st) {
  if (d->param_dtype == FCD_DT_F32) return ln_finish<float>(who, a, groups, dgamma, dbeta, accumulate, st);
  if (d->param_dtype == FCD_DT_BF16) return ln_finish<bf16_t>(who, a, groups, dgamma, dbeta, accumulate, st);
  return ln_finish<f16_t>(who, a, groups, dgamma, dbeta, accumulate, st);
}

}  // namespace

extern "C" int fcd_layernorm_desc_bytes(void) { return (int)sizeof(FcdLayerNormDesc); }

extern "C" size_t fcd_layernorm_workspace_bytes(const FcdLayerNormDesc* d) {
  if (!d || d->rows <= 0 || d->cols <= 0) return 0;
  return (size_t)ln_groups(d->rows) * 2 * (size_t)d->cols * sizeof(float);
}

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
  const dim3 grid((unsigned)(d->rows < (1 << 20) ? d->rows : (1 << 20)));
  hipStream_t st = fcd_stream(stream);
  if (d->dtype == FCD_DT_F32) ln_fwd_long<float, 1024><<<grid, 1024, 0, st>>>(a);
  else if (d->dtype == FCD_DT_BF16) ln_fwd_long<bf16_t, 1024><<<grid, 1024, 0, st>>>(a);
  else ln_fwd_long<f16_t, 1024><<<grid, 1024, 0, st>>>(a);
  return fcd_check_launch(who);
}

extern "C" int fcd_layernorm_bwd(const FcdLayerNormDesc* d, const void* gy, const void* x, const float* mean, const float* rstd,
                                 const void* gamma, const void* beta, void* dx, void* dgamma, void* dbeta, int accumulate,
                                 void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "fcd_layernorm_bwd";
  LnArgs a;
  FCD_TRY(ln_check(who, d, &a));
  const int es = fcd_dt_bytes(d->dtype);
  const RowView vx{"x", x, d->ld_x}, vg{"gy", gy, d->ld_gy}, vo{"dx", dx, d->ld_out};
  FCD_TRY(fcd_check_rows(who, vx, d->rows, d->cols, es, false));
  FCD_TRY(fcd_check_rows(who, vg, d->rows, d->cols, es, false));
  FCD_TRY(fcd_check_rows(who, vo, d->rows, d->cols, es, true));
  FCD_TRY(fcd_check_apart(who, vo, vx, d->rows, d->cols, es, true));
  FCD_TRY(fcd_check_apart(who, vo, vg, d->rows, d->cols, es, true));
  FCD_TRY(ln_check_vectors(who, d, gamma, beta, mean, rstd));
  FCD_TRY(ln_check_vectors(who, d, dgamma, dbeta, nullptr, nullptr));
  FCD_REQUIRE(d->rows == 0 || (mean && rstd), "%s: mean / rstd are NULL", who);
  const bool affine = dgamma || dbeta;
  if (affine && workspace_bytes < fcd_layernorm_workspace_bytes(d)) {
    fcd_set_error("%s: workspace of %zu bytes, needs %zu", who, workspace_bytes, fcd_layernorm_workspace_bytes(d));
    return FCD_EWORKSPACE;
  }
  FCD_REQUIRE(!affine || d->rows == 0 || (workspace && ((uintptr_t)workspace & 15u) == 0), "%s: workspace is NULL or not 16-byte aligned", who);
  a.x = x, a.gy = gy, a.gamma = gamma, a.beta = beta, a.out = dx, a.mean = (float*)mean, a.rstd = (float*)rstd;
  a.partial = affine ? (float*)workspace : nullptr;
  const int groups = (int)ln_groups(d->rows);
  hipStream_t st = fcd_stream(stream);
  if (d->rows) {
    if (d->dtype == FCD_DT_F32) ln_bwd_long<float, 1024><<<groups, 1024, 0, st>>>(a);
    else if (d->dtype == FCD_DT_BF16) ln_bwd_long<bf16_t, 1024><<<groups, 1024, 0, st>>>(a);
    else ln_bwd_long<f16_t, 1024><<<groups, 1024, 0, st>>>(a);
    FCD_TRY(fcd_check_launch(who));
  }
  return affine ? ln_finish(who, d, a, groups, dgamma, dbeta, accumulate, st) : FCD_OK;
}

extern "C" int fcd_layernorm_bwd2(const FcdLayerNormDesc* d, const void* ggx, const void* gy, const void* x, const float* mean,
                                  const float* rstd, const void* gamma, const void* beta, void* ggy, void* gx, void* dgamma,
                                  void* dbeta, int accumulate, void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "fcd_layernorm_bwd2";
  LnArgs a;
  FCD_TRY(ln_check(who, d, &a));
  const int es = fcd_dt_bytes(d->dtype);
  const RowView in[3] = {{"x", x, d->ld_x}, {"gy", gy, d->ld_gy}, {"ggx", ggx, d->ld_ggx}};
  const RowView out[2] = {{"gx", gx, d->ld_out}, {"ggy", ggy, d->ld_ggy}};
  for (const RowView& v : in) FCD_TRY(fcd_check_rows(who, v, d->rows, d->cols, es, false));
  for (const RowView& v : out) {
    FCD_TRY(fcd_check_rows(who, v, d->rows, d->cols, es, true));
    for (const RowView& w : in) FCD_TRY(fcd_check_apart(who, v, w, d->rows, d->cols, es, true));
  }
  FCD_TRY(fcd_check_apart(who, out[0], out[1], d->rows, d->cols, es, false));
  FCD_TRY(ln_check_vectors(who, d, gamma, beta, mean, rstd));
  FCD_TRY(ln_check_vectors(who, d, dgamma, dbeta, nullptr, nullptr));
  FCD_REQUIRE(d->rows == 0 || (mean && rstd), "%s: mean / rstd are NULL", who);
  const bool affine = dgamma || dbeta;
  if (affine && workspace_bytes < fcd_layernorm_workspace_bytes(d)) {
    fcd_set_error("%s: workspace of %zu bytes, needs %zu", who, workspace_bytes, fcd_layernorm_workspace_bytes(d));
    return FCD_EWORKSPACE;
  }
  FCD_REQUIRE(!affine || d->rows == 0 || (workspace && ((uintptr_t)workspace & 15u) == 0), "%s: workspace is NULL or not 16-byte aligned", who);
  a.x = x, a.gy = gy, a.ggx = ggx, a.gamma = gamma, a.beta = beta, a.out = gx, a.ggy = ggy;
  a.mean = (float*)mean, a.rstd = (float*)rstd;
  a.partial = affine ? (float*)workspace : nullptr;
  const int groups = (int)ln_groups(d->rows);
  hipStream_t st = fcd_stream(stream);
  if (d->rows) {
    if (d->dtype == FCD_DT_F32) ln_bwd2_long<float, 1024><<<groups, 1024, 0, st>>>(a);
    else if (d->dtype == FCD_DT_BF16) ln_bwd2_long<bf16_t, 1024><<<groups, 1024, 0, st>>>(a);
    else ln_bwd2_long<f16_t, 1024><<<groups, 1024, 0, st>>>(a);
    FCD_TRY(fcd_check_launch(who));
  }
  return affine ? ln_finish(who, d, a, groups, dgamma, dbeta, accumulate, st) : FCD_OK;
}
