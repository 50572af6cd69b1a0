// Layer norm: argument checks, scratch, and the last step of the affine gradients, shared by its directions.
#include "fcd_layernorm.h"

namespace {

// dgamma (blockIdx.y 0) / dbeta (1): the workgroups' sums of a column, added in 2^ls strands and joined in order.  Up to 32
// strands of 16 columns (64-byte accesses) where there are many sums, down to one strand of 512 columns.  256 sums of 4096
// columns 4.4 us, most of it the launch; 8 of 262144 9.6 (28 with 32 strands).
template <typename P>
__global__ __launch_bounds__(512) void ln_affine_reduce(const float* partial, int groups, long cols, int ls, P* dgamma, P* dbeta,
                                                        int accumulate) {
  __shared__ float sm[512];
  P* out = blockIdx.y ? dbeta : dgamma;
  if (!out) return;
  const int strands = 1 << ls, width = 512 >> ls, col = threadIdx.x & (width - 1), strand = threadIdx.x >> (9 - ls);
  const long c = (long)blockIdx.x * width + col;
  float s = 0.f;
  if (c < cols)
#pragma unroll 4
    for (int g = strand; g < groups; g += strands) s += partial[((long)g * 2 + blockIdx.y) * cols + c];
  sm[threadIdx.x] = s;
  __syncthreads();
  if (strand == 0 && c < cols) {
    s = 0.f;
    for (int i = 0; i < strands; ++i) s += sm[i * width + col];
    out[c] = (P)(accumulate ? (float)out[c] + s : s);
  }
}

template <typename P>
int reduce(const char* who, const LnArgs& a, int groups, void* dgamma, void* dbeta, int accumulate, hipStream_t st) {
  int ls = 0;
  while (ls < 5 && (1 << ls) < groups) ++ls;
  const long width = 512 >> ls;
  ln_affine_reduce<P><<<dim3((unsigned)((a.cols + width - 1) / width), 2), 512, 0, st>>>(a.partial, groups, a.cols, ls, (P*)dgamma,
                                                                                        (P*)dbeta, accumulate);
  return fcd_check_launch(who);
}

}  // namespace

int ln_groups(int64_t rows, int64_t cols) {
  const LnShape s = ln_bwd_shape(cols);
  const int64_t rpb = s.g > 0 && s.g <= 64 ? 256 / s.g : 1, need = (rows + rpb - 1) / rpb;
  int64_t full;
  if (s.g == 0) {            // split rows: enough workgroups of 2048 columns for the card, and not more than 256 sums of a column
    full = 2048 / ((cols + 2047) / 2048);
    full = full < 1 ? 1 : full > 256 ? 256 : full;
  } else {
    // Every workgroup's sums are written and read once more: 512 threads a compute unit, twice that where a workgroup has 128.
    // Twice as many: 4096 x 4096 bf16 31 -> 35 us and its join 4.5 -> 6.8, with an activation 38 -> 36 and 4.5 -> 6.7;
    // 65536 x 64 fp32 17.6 either way, its join 4.2 -> 5.0.
    full = s.g <= 64 ? 512 : s.g >= 512 ? 256 : 256 * 512 / s.g;
  }
  return (int)(need < full ? need : full);
}

bool ln_few_rows(int64_t rows, int64_t cols) {
  const LnShape s = ln_bwd_shape(cols);
  return s.g && rows > 0 && rows <= (s.g > 256 ? s.g : 256) / 2;   // four turns of a column workgroup
}

int ln_finish(const char* who, const FcdLayerNormDesc* d, const LnArgs& a, int groups, void* dgamma, void* dbeta, int accumulate,
              hipStream_t st) {
  if (d->param_dtype == FCD_DT_F32) return reduce<float>(who, a, groups, dgamma, dbeta, accumulate, st);
  if (d->param_dtype == FCD_DT_BF16) return reduce<bf16_t>(who, a, groups, dgamma, dbeta, accumulate, st);
  return reduce<f16_t>(who, a, groups, dgamma, dbeta, accumulate, st);
}

namespace {

// Scratch of one pass, in floats from its start: affine sums, chunk sums, row sums.
struct Scratch {
  size_t chunk, row, bytes;
};

Scratch scratch(const FcdLayerNormDesc* d, int pass, bool affine) {
  Scratch s = {};
  if (d->rows <= 0 || d->cols <= 0) return s;
  const size_t rows = (size_t)d->rows, cols = (size_t)d->cols;
  const bool split = pass == FCD_LN_FWD ? d->cols > LN_FWD_MAX : ln_bwd_shape(d->cols).g == 0;
  if (pass != FCD_LN_FWD && affine && !(pass == FCD_LN_BWD && ln_few_rows(d->rows, d->cols)))
    s.chunk = (size_t)ln_groups(d->rows, d->cols) * 2 * cols;
  s.row = s.chunk;
  s.bytes = s.chunk * sizeof(float);
  if (split) {
    s.row += rows * (size_t)ln_chunks(d->cols) * (pass == FCD_LN_BWD2 ? 5 : 2);
    s.bytes = (s.row + rows * (pass == FCD_LN_FWD ? 2 : ROW_SUMS)) * sizeof(float);
  }
  return s;
}

}  // namespace

int ln_check_scratch(const char* who, const FcdLayerNormDesc* d, int pass, const void* dgamma, const void* dbeta, void* workspace,
                     size_t workspace_bytes, LnArgs* a) {
  FCD_TRY(ln_check_vectors(who, d, dgamma, dbeta, nullptr, nullptr));
  const bool affine = dgamma || dbeta;
  const Scratch s = scratch(d, pass, affine);
  if (workspace_bytes < s.bytes) {
    fcd_set_error("%s: workspace of %zu bytes, needs %zu", who, workspace_bytes, s.bytes);
    return FCD_EWORKSPACE;
  }
  FCD_REQUIRE(s.bytes == 0 || (workspace && ((uintptr_t)workspace & 15u) == 0), "%s: workspace is NULL or not 16-byte aligned", who);
  if (s.chunk) a->partial = (float*)workspace;
  a->chunk = (float*)workspace + s.chunk;
  a->row = (float*)workspace + s.row;
  return FCD_OK;
}

int ln_check(const char* who, const FcdLayerNormDesc* d, LnArgs* a) {
  FCD_REQUIRE(d, "%s: NULL descriptor", who);
  FCD_REQUIRE(fcd_dt_bytes(d->dtype), "%s: unknown element type %d", who, d->dtype);
  FCD_REQUIRE(d->param_dtype == FCD_DT_F32 || d->param_dtype == d->dtype, "%s: parameters must be fp32 or of x's type", who);
  FCD_REQUIRE(d->rows >= 0, "%s: negative number of rows", who);
  FCD_REQUIRE(d->cols >= 1 && d->cols <= (int64_t)1 << 30, "%s: %lld columns (1 ... 2^30)", who, (long long)d->cols);
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

int ln_check_apart(const char* who, const FcdLayerNormDesc* d, const Bytes* w, int nw, const Bytes* r, int nr, const RowView* t,
                   int nt) {
  const int es = fcd_dt_bytes(d->dtype);
  for (int i = 0; i < nw; ++i) {
    for (int k = i + 1; k < nw; ++k) FCD_TRY(fcd_check_apart(who, w[i], w[k]));
    for (int k = 0; k < nr; ++k) FCD_TRY(fcd_check_apart(who, w[i], r[k]));
    for (int k = 0; k < nt; ++k) FCD_TRY(fcd_check_apart(who, w[i], t[k], d->rows, d->cols, es));
  }
  return FCD_OK;
}

extern "C" int fcd_layernorm_desc_bytes(void) { return (int)sizeof(FcdLayerNormDesc); }

extern "C" size_t fcd_layernorm_workspace_bytes(const FcdLayerNormDesc* d, int pass, int affine) {
  return d && pass >= FCD_LN_FWD && pass <= FCD_LN_BWD2 ? scratch(d, pass, affine != 0).bytes : 0;
}
