// Layer norm backward: dx, and the row sums of the affine gradients.
#include "fcd_layernorm.h"

namespace {

// A row's x and gy in registers, one exchange for both of its sums, dx out; a thread meets the same columns in every row, so
// the affine sums stay in its registers until the last row.  The next row's loads are in flight meanwhile.  One unit of 8
// columns a thread leaves the registers for it (1024 threads are four waves a SIMD, shorter rows get two: ln_groups); two units,
// two waves and no prefetch took 244 us for 16384 x 8192 bf16 dropout where one took 174 (141 to 188 now, by the process).
// Bound by memory, 16384 x 8192 bf16 146 us (5.5 TB/s), 4096 x 4096 19.3, 65536 x 64 fp32 10.2 (with dropout the
// vector ALU is 67 % active at 16384 x 8192).  The affine join behind it: 4 to 7 us.
// EPI 0: plain; 1: dropout; 2: activation, and dropout if there is any.
// (`blocks` workgroups from the first on; AFFINE: the affine sums are kept.)
template <typename T, int G, int NV, int EPI, bool AFFINE>
__device__ __forceinline__ void bwd_rows(LnArgs p, unsigned blocks) {
  constexpr int TH = G > 64 ? G : 256, RPB = TH / G, WAVES = RowSums<G, 2>::WAVES;
  __shared__ float sm[2 * 2 * WAVES];
  int turn = 0;
  if (EPI) drop_state(p.drop);
  const int lane = threadIdx.x % G, cols = (int)p.cols;
  const float inv = 1.f / (float)cols;
  float ga[NV][8], be[NV][8], dg[NV][8], db[NV][8];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (lane + k * G) * 8;
    load_param<T>(p.gamma, p.param_f32, c, cols - c, 1.f, ga[k]);
    if (EPI == 2) load_param<T>(p.beta, p.param_f32, c, cols - c, 0.f, be[k]);
#pragma unroll
    for (int j = 0; j < 8; ++j) dg[k][j] = db[k][j] = 0.f;
  }
  typename Oct<T>::type nx[NV], ng[NV];
  float nmean = 0.f, nrstd = 0.f;
  auto fetch = [&](long r) {
    const bool here = G >= 64 || r < p.rows;
    nmean = here ? p.mean[r] : 0.f;
    nrstd = here ? p.rstd[r] : 0.f;
    const T *x = (const T*)p.x + r * p.ld_x, *gy = (const T*)p.gy + r * p.ld_gy;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (lane + k * G) * 8;
      if (here) {
        fetch8<T, G>(x, c, cols, nx[k]);
        fetch8<T, G>(gy, c, cols, ng[k]);
      }
    }
  };
  // G < 64: every thread of a wave makes the same number of turns, for the sums need whole groups; G >= 64: whole waves do
  long row = first_row<G, TH>();
  const long step = (long)blocks * RPB;
  long turns = (p.rows - (G >= 64 ? row : (long)blockIdx.x * RPB) + step - 1) / step;
  if (idle_wave<G>(cols)) {
    for (; turns > 0; --turns) idle_sums<G, 2>(sm, turn);
  }
  if (turns > 0) fetch(row);
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    arrive<T>(nx[k]);
    arrive<T>(ng[k]);
  }
  for (long it = 0; it < turns; ++it, row += step) {
    const float mean = nmean, rstd = nrstd;
    float xh[NV][8], a[NV][8];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int n = G >= 64 || row < p.rows ? cols - (lane + k * G) * 8 : 0;
      settle<T, G>(nx[k], cols, n);
      settle<T, G>(ng[k], cols, n);
      widen<T>(nx[k], xh[k]);
      widen<T>(ng[k], a[k]);
    }
    if (it + 1 < turns) fetch(row + step);
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (EPI && p.drop.t) {
        uint32_t w[4];
        drop_draw8(p.drop, (uint64_t)(row * cols + (lane + k * G) * 8), w);
        drop_apply(p.drop, w, a[k]);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) xh[k][j] = (xh[k][j] - mean) * rstd;      // (absent elements: gy is 0, and so is what follows)
      if (EPI == 2) {
        float u[8], d1[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] = fmaf(xh[k][j], ga[k][j], be[k][j]);
        ln_act8(u, p.act, nullptr, d1, nullptr);
#pragma unroll
        for (int j = 0; j < 8; ++j) a[k][j] *= d1[j];
      }
      float s0 = 0.f, s1 = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float g1 = a[k][j];
        if (AFFINE) {
          dg[k][j] = fmaf(g1, xh[k][j], dg[k][j]);
          db[k][j] += g1;
        }
        a[k][j] = g1 * ga[k][j];
        s0 += a[k][j];
        s1 = fmaf(a[k][j], xh[k][j], s1);
      }
      s[0] += s0;
      s[1] += s1;
    }
    RowSums<G, 2>::run(s, sm, turn);
    const float c0 = -rstd * (s[0] * inv), c1 = -rstd * (s[1] * inv);
    T* out = (T*)p.out + row * p.ld_out;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
#pragma unroll
      for (int j = 0; j < 8; ++j) a[k][j] = fmaf(a[k][j], rstd, fmaf(xh[k][j], c1, c0));
      arrive<T>(nx[k]);
      arrive<T>(ng[k]);
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (lane + k * G) * 8, n = G >= 64 || row < p.rows ? cols - c : 0;
      store8(out + c, n, a[k]);
    }
  }
  if constexpr (AFFINE) {
    __shared__ float aff[affine_lds<G, NV>()];
    if (p.partial) write_partial<G, NV>(p, dg, db, aff);
  }
}

template <typename T, int G, int NV, int EPI>
__global__ __launch_bounds__(G > 64 ? G : 256) void ln_bwd_rows(LnArgs p) {
  bwd_rows<T, G, NV, EPI, true>(p, gridDim.x);
}

struct Affine {
  void *dgamma, *dbeta;
  int accumulate;
};

template <typename T>
__device__ __forceinline__ void put_affine(void* out, int f32, int accumulate, int c, float v) {
  if (!out) return;
  if (f32) {
    float* o = (float*)out + c;
    *o = accumulate ? *o + v : v;
  } else {
    T* o = (T*)out + c;
    *o = (T)(accumulate ? (float)*o + v : v);
  }
}

// Few rows: the first `blocks` workgroups write dx; the others sum 64 columns each over all rows, which needs nothing from the
// first ones (the row sums do not enter the affine gradients).  x and gy are read twice, from cache; in exchange there is
// no scratch and no second launch: 64 x 2048 fp32 8.4 -> 4.8 us, 128 x 8192 bf16 12.8 -> 5.7.  Up to four turns of a column
// workgroup: 512 x 2048 (sixteen) takes 10.4 us here and 12.4 in two launches, 256 x 1024 with an activation 12.8 and 8.9.
template <typename T, int G, int EPI>
__global__ __launch_bounds__(G > 64 ? G : 256) void ln_bwd_few(LnArgs p, Affine f, unsigned blocks) {
  constexpr int TH = G > 64 ? G : 256;
  if (blockIdx.x < blocks) {
    bwd_rows<T, G, 1, EPI, false>(p, blocks);
    return;
  }
  __shared__ float sm[TH / 64][8][16];
  if (EPI) drop_state(p.drop);
  const int unit = threadIdx.x & 7, cols = (int)p.cols, c = ((int)(blockIdx.x - blocks) * 8 + unit) * 8, n = cols - c;
  float ga[8], be[8], dg[8], db[8];
  if (EPI == 2) {
    load_param<T>(p.gamma, p.param_f32, c, n, 1.f, ga);
    load_param<T>(p.beta, p.param_f32, c, n, 0.f, be);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) dg[j] = db[j] = 0.f;
  for (long row = threadIdx.x >> 3; row < p.rows; row += TH / 8) {
    const float mean = p.mean[row], rstd = p.rstd[row];
    float xh[8], g[8];
    load8((const T*)p.x + row * p.ld_x + c, n, xh);
    load8((const T*)p.gy + row * p.ld_gy + c, n, g);
    if (EPI && p.drop.t) {
      uint32_t w[4];
      drop_draw8(p.drop, (uint64_t)(row * cols + c), w);
      drop_apply(p.drop, w, g);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) xh[j] = (xh[j] - mean) * rstd;
    if (EPI == 2) {
      float u[8], d1[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) u[j] = fmaf(xh[j], ga[j], be[j]);
      ln_act8(u, p.act, nullptr, d1, nullptr);
#pragma unroll
      for (int j = 0; j < 8; ++j) g[j] *= d1[j];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      dg[j] = fmaf(g[j], xh[j], dg[j]);
      db[j] += g[j];
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
#pragma unroll
    for (int o = 8; o < 64; o <<= 1) {
      dg[j] += __shfl_xor(dg[j], o, 64);
      db[j] += __shfl_xor(db[j], o, 64);
    }
    if ((threadIdx.x & 63) < 8) {
      sm[threadIdx.x >> 6][unit][j] = dg[j];
      sm[threadIdx.x >> 6][unit][8 + j] = db[j];
    }
  }
  __syncthreads();
  if (threadIdx.x < 128) {
    const int which = threadIdx.x >> 6, i = threadIdx.x & 63, col = (int)(blockIdx.x - blocks) * 64 + i;
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < TH / 64; ++w) s += sm[w][i >> 3][which * 8 + (i & 7)];
    if (col < cols) put_affine<T>(which ? f.dbeta : f.dgamma, p.param_f32, f.accumulate, col, s);
  }
}

// Split rows, 1: a chunk's two sums.  All four kernels: 4096 x 12288 bf16 115 us (one workgroup per row that read it again and
// kept the affine sums in memory: 416), 8 x 262144 fp32 29 (348).
template <typename T, int EPI>
__global__ __launch_bounds__(256) void ln_bwd_chunks(LnArgs p, long chunks) {
  __shared__ float sm[2 * 2 * 4];
  int turn = 0;
  if (EPI) drop_state(p.drop);
  for (long item = blockIdx.x; item < p.rows * chunks; item += gridDim.x) {
    const long row = item / chunks, c0 = (item - row * chunks) * CHUNK;
    const T *x = (const T*)p.x + row * p.ld_x, *gy = (const T*)p.gy + row * p.ld_gy;
    const float mean = p.mean[row], rstd = p.rstd[row];
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int c = (int)c0 + (threadIdx.x + k * 256) * 8, n = (int)p.cols - c;
      Eight<EPI, false> e;
      float ga[8], be[8];
      load8(x + c, n, e.xh);
      load8(gy + c, n, e.g);
      load_param<T>(p.gamma, p.param_f32, c, n, 1.f, ga);
      if (EPI == 2) load_param<T>(p.beta, p.param_f32, c, n, 0.f, be);
      e.make(p, row, c, mean, rstd, ga, be);
      float s0 = 0.f, s1 = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float a = (EPI == 2 ? e.g[j] * e.d1[j] : e.g[j]) * ga[j];
        s0 += a;
        s1 = fmaf(a, e.xh[j], s1);
      }
      s[0] += s0;
      s[1] += s1;
    }
    RowSums<256, 2>::run(s, sm, turn);
    if (threadIdx.x == 0) {
      p.chunk[item * 2] = s[0];
      p.chunk[item * 2 + 1] = s[1];
    }
  }
}

// 3 (2 is ln_join): dx and the affine sums of a row group.
template <typename T, int EPI>
__global__ __launch_bounds__(256) void ln_bwd_stream(LnArgs p) {
  if (EPI) drop_state(p.drop);
  const int c = (int)((blockIdx.x * 256u + threadIdx.x) * 8), cols = (int)p.cols, n = cols - c;
  if (n <= 0) return;
  const float inv = 1.f / (float)cols;
  float ga[8], be[8], dg[8], db[8];
  load_param<T>(p.gamma, p.param_f32, c, n, 1.f, ga);
  if (EPI == 2) load_param<T>(p.beta, p.param_f32, c, n, 0.f, be);
#pragma unroll
  for (int j = 0; j < 8; ++j) dg[j] = db[j] = 0.f;
  typename Oct<T>::type nx, ng;
  long row = blockIdx.y;
  fetch8<T, 64>((const T*)p.x + row * p.ld_x, c, cols, nx);
  fetch8<T, 64>((const T*)p.gy + row * p.ld_gy, c, cols, ng);
  arrive<T>(nx);
  arrive<T>(ng);
  for (; row < p.rows; row += gridDim.y) {
    settle<T, 64>(nx, cols, n);
    settle<T, 64>(ng, cols, n);
    Eight<EPI, false> e;
    widen<T>(nx, e.xh);
    widen<T>(ng, e.g);
    const long next = row + gridDim.y;
    if (next < p.rows) {
      fetch8<T, 64>((const T*)p.x + next * p.ld_x, c, cols, nx);
      fetch8<T, 64>((const T*)p.gy + next * p.ld_gy, c, cols, ng);
    }
    const float mean = p.mean[row], rstd = p.rstd[row];
    const float c0 = -rstd * (p.row[row * ROW_SUMS] * inv), c1 = -rstd * (p.row[row * ROW_SUMS + 1] * inv);
    e.make(p, row, c, mean, rstd, ga, be);
    float dx[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float g1 = EPI == 2 ? e.g[j] * e.d1[j] : e.g[j];
      dg[j] = fmaf(g1, e.xh[j], dg[j]);
      db[j] += g1;
      dx[j] = fmaf(g1 * ga[j], rstd, fmaf(e.xh[j], c1, c0));
    }
    arrive<T>(nx);
    arrive<T>(ng);
    store8((T*)p.out + row * p.ld_out + c, n, dx);
  }
  if (p.partial) {
    float* part = p.partial + (long)blockIdx.y * 2 * cols + c;
    store8(part, n, dg);
    store8(part + cols, n, db);
  }
}

template <typename T, int EPI>
void launch_split(const LnArgs& a, hipStream_t st) {
  const long chunks = ln_chunks(a.cols);
  ln_bwd_chunks<T, EPI><<<ln_items(a.rows, a.cols), 256, 0, st>>>(a, chunks);
  ln_join<2><<<ln_join_grid(a.rows), 256, 0, st>>>(a.chunk, a.rows, chunks, a.row, 0);
  ln_bwd_stream<T, EPI><<<ln_stream_grid(a.rows, a.cols), 256, 0, st>>>(a);
}

template <typename T>
void launch(const LnArgs& a, int groups, hipStream_t st) {
  const LnShape s = ln_bwd_shape(a.cols);
  if (s.g == 0) {
    if (a.act != 1.f) launch_split<T, 2>(a, st);
    else if (a.drop.t) launch_split<T, 1>(a, st);
    else launch_split<T, 0>(a, st);
    return;
  }
#define SHAPE(G, NV)                                                                                      \
  if (s.g == G && s.nv == NV) {                                                                           \
    if (a.act != 1.f) ln_bwd_rows<T, G, NV, 2><<<groups, G > 64 ? G : 256, 0, st>>>(a);                     \
    else if (a.drop.t) ln_bwd_rows<T, G, NV, 1><<<groups, G > 64 ? G : 256, 0, st>>>(a);                    \
    else ln_bwd_rows<T, G, NV, 0><<<groups, G > 64 ? G : 256, 0, st>>>(a);                                  \
  }
  LN_BWD_SHAPES(SHAPE)
#undef SHAPE
}

template <typename T>
void launch_few(const LnArgs& a, const Affine& f, int groups, hipStream_t st) {
  const LnShape s = ln_bwd_shape(a.cols);
  const unsigned grid = groups + (unsigned)((a.cols + 63) / 64);
#define SHAPE(G, NV)                                                                                      \
  if (s.g == G) {                                                                                         \
    if (a.act != 1.f) ln_bwd_few<T, G, 2><<<grid, G > 64 ? G : 256, 0, st>>>(a, f, groups);               \
    else if (a.drop.t) ln_bwd_few<T, G, 1><<<grid, G > 64 ? G : 256, 0, st>>>(a, f, groups);              \
    else ln_bwd_few<T, G, 0><<<grid, G > 64 ? G : 256, 0, st>>>(a, f, groups);                            \
  }
  LN_BWD_SHAPES(SHAPE)
#undef SHAPE
}

}  // namespace

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
  FCD_REQUIRE(d->rows == 0 || (mean && rstd), "%s: mean / rstd are NULL", who);
  FCD_TRY(ln_check_scratch(who, d, FCD_LN_BWD, dgamma, dbeta, workspace, workspace_bytes, &a));
  const int64_t ps = fcd_dt_bytes(d->param_dtype) * d->cols, ss = 4 * d->rows;
  const Bytes written[] = {{"dgamma", dgamma, ps}, {"dbeta", dbeta, ps}, {"workspace", workspace, (int64_t)workspace_bytes}};
  const Bytes read[] = {{"mean", mean, ss}, {"rstd", rstd, ss}, {"gamma", gamma, ps}, {"beta", beta, ps}, {"rng", d->rng, 16}};
  const RowView rows[] = {vx, vg, vo};
  FCD_TRY(ln_check_apart(who, d, written, 3, read, 5, rows, 3));
  for (const Bytes& b : read) FCD_TRY(fcd_check_apart(who, b, vo, d->rows, d->cols, es));
  a.x = x, a.gy = gy, a.gamma = gamma, a.beta = beta, a.out = dx, a.mean = (float*)mean, a.rstd = (float*)rstd;
  const int groups = ln_groups(d->rows, d->cols);
  hipStream_t st = fcd_stream(stream);
  const bool few = (dgamma || dbeta) && ln_few_rows(d->rows, d->cols);
  const bool in_place = dx == gy || dx == x;   // dx would overwrite what the column workgroups read: those go first
  if (few) {
    const Affine f{dgamma, dbeta, accumulate};
    const int beside = in_place ? 0 : groups;
    if (d->dtype == FCD_DT_F32) launch_few<float>(a, f, beside, st);
    else if (d->dtype == FCD_DT_BF16) launch_few<bf16_t>(a, f, beside, st);
    else launch_few<f16_t>(a, f, beside, st);
    FCD_TRY(fcd_check_launch(who));
    if (!in_place) return FCD_OK;
  }
  if (d->rows) {
    if (d->dtype == FCD_DT_F32) launch<float>(a, groups, st);
    else if (d->dtype == FCD_DT_BF16) launch<bf16_t>(a, groups, st);
    else launch<f16_t>(a, groups, st);
    FCD_TRY(fcd_check_launch(who));
  }
  return (dgamma || dbeta) && !few ? ln_finish(who, d, a, groups, dgamma, dbeta, accumulate, st) : FCD_OK;
}

