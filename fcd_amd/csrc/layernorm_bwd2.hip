// Layer norm: backward of the backward pass (the cotangents of gy and x for one of dx), for gradient penalties.
#include "fcd_layernorm.h"

namespace {

// A row's x, gy and v = ggx in registers; the four means in one exchange, then S = mean((v - mean v - xhat mean(v xhat)) (a -
// mean a)) and behind a curved activation the two sums of q gamma in a second one.  (S in the first exchange, as mean(v a) less
// the products of the means, loses the square of the gradients' offsets.  The second exchange costs 0 to 3 %; 4096 x 4095 40 ->
// 44 us, 2048 x 8192 behind a leaky slope 37.7 -> 39.7.  Waves that centre on their own means and join them in the first one:
// equal or slower, and spilt.)
// With the row's sums in hand gx is a combination of four things: c0 + c1 t + c2 a + c3 xhat (+ rstd q gamma).
// Bound by memory without an activation, 16384 x 8192 bf16 245 us (5.5 TB/s), 4096 x 4096 29, 65536 x 64 fp32 16; with SiLU and
// dropout by the vector ALU (79 % active at 4096 x 4096 bf16, 39 to 41 us).  Four waves a SIMD by force spill: 65536 x 64 fp32 SiLU
// 17.6 -> 34.6 us.
// EPI 0: plain; 1: dropout; 2: activation, and dropout if there is any.
template <typename T, int G, int NV, int EPI>
__global__ __launch_bounds__(G > 64 ? G : 256) void ln_bwd2_rows(LnArgs p) {
  constexpr int TH = G > 64 ? G : 256, RPB = TH / G, WAVES = RowSums<G, 4>::WAVES;
  __shared__ float sm[2 * 4 * WAVES], sm2[2 * (EPI == 2 ? 3 : 1) * WAVES];
  __shared__ float aff[affine_lds<G, NV>()];
  int turn = 0, turn2 = 0;
  if (EPI) drop_state(p.drop);
  const int lane = threadIdx.x % G, cols = (int)p.cols;
  const float inv = 1.f / (float)cols;
  const bool curved = EPI == 2 && p.act > 1.f;
  float ga[NV][8], be[NV][8], dg[NV][8], db[NV][8];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (lane + k * G) * 8;
    load_param<T>(p.gamma, p.param_f32, c, cols - c, 1.f, ga[k]);
    if (EPI == 2) load_param<T>(p.beta, p.param_f32, c, cols - c, 0.f, be[k]);
#pragma unroll
    for (int j = 0; j < 8; ++j) dg[k][j] = db[k][j] = 0.f;
  }
  typename Oct<T>::type nx[NV], ng[NV], nv[NV];
  float nmean = 0.f, nrstd = 0.f;
  auto fetch = [&](long r) {
    const bool here = G >= 64 || r < p.rows;
    nmean = here ? p.mean[r] : 0.f;
    nrstd = here ? p.rstd[r] : 0.f;
    const T *x = (const T*)p.x + r * p.ld_x, *gy = (const T*)p.gy + r * p.ld_gy, *v = (const T*)p.ggx + r * p.ld_ggx;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (lane + k * G) * 8;
      if (here) {
        fetch8<T, G>(x, c, cols, nx[k]);
        fetch8<T, G>(gy, c, cols, ng[k]);
        fetch8<T, G>(v, c, cols, nv[k]);
      }
    }
  };
  // G < 64: every thread of a wave makes the same number of turns, for the sums need whole groups; G >= 64: whole waves do
  long row = first_row<G, TH>();
  const long step = (long)gridDim.x * RPB;
  long turns = (p.rows - (G >= 64 ? row : (long)blockIdx.x * RPB) + step - 1) / step;
  if (idle_wave<G>(cols)) {
    for (; turns > 0; --turns) {
      idle_sums<G, 4>(sm, turn);
      if (curved) idle_sums<G, 3>(sm2, turn2);
      else idle_sums<G, 1>(sm2, turn2);
    }
  }
  // a workgroup of 1024 has 128 registers a thread: behind an activation they do not hold the next row as well
  constexpr bool AHEAD = !(G == 1024 && EPI == 2);
  if (AHEAD && turns > 0) fetch(row);
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    if (AHEAD) {
      arrive<T>(nx[k]);
      arrive<T>(ng[k]);
      arrive<T>(nv[k]);
    }
  }
  for (long it = 0; it < turns; ++it, row += step) {
    if (!AHEAD) fetch(row);
    const float mean = nmean, rstd = nrstd;
    // xhat, drop(gy), v, and behind an activation act'(u) and act''(u)
    float xh[NV][8], g[NV][8], v[NV][8], d1[NV][8], q[NV][8], s[4] = {0.f, 0.f, 0.f, 0.f};
    uint32_t w[NV][4];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int n = G >= 64 || row < p.rows ? cols - (lane + k * G) * 8 : 0;
      settle<T, G>(nx[k], cols, n);
      settle<T, G>(ng[k], cols, n);
      settle<T, G>(nv[k], cols, n);
      widen<T>(nx[k], xh[k]);
      widen<T>(ng[k], g[k]);
      widen<T>(nv[k], v[k]);
    }
    if (AHEAD && it + 1 < turns) fetch(row + step);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (EPI && p.drop.t) {
        drop_draw8(p.drop, (uint64_t)(row * cols + (lane + k * G) * 8), w[k]);
        drop_apply(p.drop, w[k], g[k]);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) xh[k][j] = (xh[k][j] - mean) * rstd;      // (absent elements: gy and v are 0)
      if (EPI == 2) {
        float u[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] = fmaf(xh[k][j], ga[k][j], be[k][j]);
        ln_act8(u, p.act, nullptr, d1[k], q[k]);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          q[k][j] *= g[k][j] * ga[k][j];
          g[k][j] *= d1[k][j];                        // g1
        }
      }
      float t[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float a = g[k][j] * ga[k][j];
        t[0] += a;
        t[1] = fmaf(a, xh[k][j], t[1]);
        t[2] += v[k][j];
        t[3] = fmaf(v[k][j], xh[k][j], t[3]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i] += t[i];
    }
    RowSums<G, 4>::run(s, sm, turn);
    const float am = s[0] * inv, ax = s[1] * inv, vm = s[2] * inv, vx = s[3] * inv;
    // t, the cotangent of a, in the place of v
    float ts = 0.f, q0 = 0.f, q1 = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int n = cols - (lane + k * G) * 8;
      float ac[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) ac[j] = fmaf(g[k][j], ga[k][j], -am);
      if (n < 8) {
#pragma unroll
        for (int j = 0; j < 8; ++j) ac[j] = j < n ? ac[j] : 0.f;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float w = v[k][j] - vm - xh[k][j] * vx;
        ts = fmaf(w, ac[j], ts);
        v[k][j] = rstd * w;
        if (EPI == 2) {
          q[k][j] *= v[k][j];
          const float qg = q[k][j] * ga[k][j];
          q0 += qg;
          q1 = fmaf(qg, xh[k][j], q1);
        }
      }
    }
    if (EPI == 2 && curved) {
      float s2[3] = {ts, q0, q1};
      RowSums<G, 3>::run(s2, sm2, turn2);
      ts = s2[0], q0 = s2[1], q1 = s2[2];
    } else {
      float s2[1] = {ts};
      RowSums<G, 1>::run(s2, sm2, turn2);
      ts = s2[0];
    }
    // with v = t / rstd + mean(v) + xhat mean(v xhat) put into h:
    const float c0 = rstd * (rstd * am * vx - q0 * inv), c1 = -rstd * ax, c2 = -rstd * rstd * vx;
    const float c3 = -rstd * (q1 * inv + rstd * (ts * inv - vx * ax));
    T *ggy = (T*)p.ggy + row * p.ld_ggy, *out = (T*)p.out + row * p.ld_out;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (lane + k * G) * 8, n = G >= 64 || row < p.rows ? cols - c : 0;
      float gg[8], gx[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        gg[j] = (EPI == 2 ? d1[k][j] * ga[k][j] : ga[k][j]) * v[k][j];
        gx[j] = fmaf(v[k][j], c1, fmaf(g[k][j] * ga[k][j], c2, fmaf(xh[k][j], c3, c0)));
        dg[k][j] = fmaf(g[k][j], v[k][j], dg[k][j]);  // (absent elements: g1 and q are 0)
        if (EPI == 2) {
          gx[j] = fmaf(q[k][j] * ga[k][j], rstd, gx[j]);
          dg[k][j] = fmaf(q[k][j], xh[k][j], dg[k][j]);
          db[k][j] += q[k][j];
        }
      }
      if (EPI && p.drop.t) drop_apply(p.drop, w[k], gg);
      if (AHEAD) {
        arrive<T>(nx[k]);
        arrive<T>(ng[k]);
        arrive<T>(nv[k]);
      }
      if (n >= 8) {
        typename Oct<T>::type o, r;
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = (T)gg[j], r[j] = (T)gx[j];
        *(typename Oct<T>::type*)(ggy + c) = o;
        *(typename Oct<T>::type*)(out + c) = r;
      } else {
        store8(ggy + c, n, gg);
        store8(out + c, n, gx);
      }
    }
  }
  if (p.partial) write_partial<G, NV>(p, dg, db, aff);
}

// Split rows, 1: a chunk's sums of a, a xhat, v and v xhat, and that of (v - its mean) (a - its mean) around the chunk's own
// means; with the joined ones known and a curved activation (CURVED) the two sums of q gamma.
// All kernels of a call: 4096 x 12288 bf16 214 us (one workgroup per row that read it again: 489), 8 x 262144 fp32 32.
template <typename T, int EPI, bool CURVED>
__global__ __launch_bounds__(256) void ln_bwd2_chunks(LnArgs p, long chunks) {
  constexpr int K = CURVED ? 2 : 5;
  __shared__ float sm[2 * 4 * 4], sm2[2 * 4];
  int turn = 0, turn2 = 0;
  if (EPI) drop_state(p.drop);
  const float inv = 1.f / (float)p.cols;
  for (long item = blockIdx.x; item < p.rows * chunks; item += gridDim.x) {
    const long row = item / chunks, c0 = (item - row * chunks) * CHUNK;
    const T *x = (const T*)p.x + row * p.ld_x, *gy = (const T*)p.gy + row * p.ld_gy, *ggx = (const T*)p.ggx + row * p.ld_ggx;
    const float mean = p.mean[row], rstd = p.rstd[row];
    const float vm = CURVED ? p.row[row * ROW_SUMS + 2] * inv : 0.f, vx = CURVED ? p.row[row * ROW_SUMS + 3] * inv : 0.f;
    float s[CURVED ? 2 : 4] = {}, a[4][8], v[4][8];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int c = (int)c0 + (threadIdx.x + k * 256) * 8, n = (int)p.cols - c;
      Eight<EPI, CURVED> e;
      float ga[8], be[8];
      load8(x + c, n, e.xh);
      load8(gy + c, n, e.g);
      load8(ggx + c, n, v[k]);
      load_param<T>(p.gamma, p.param_f32, c, n, 1.f, ga);
      if (EPI == 2) load_param<T>(p.beta, p.param_f32, c, n, 0.f, be);
      e.make(p, row, c, mean, rstd, ga, be);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if constexpr (CURVED) {
          const float qg = e.g[j] * e.d2[j] * ga[j] * (rstd * (v[k][j] - vm - e.xh[j] * vx)) * ga[j];
          s[0] += qg;
          s[1] = fmaf(qg, e.xh[j], s[1]);
        } else {
          a[k][j] = (EPI == 2 ? e.g[j] * e.d1[j] : e.g[j]) * ga[j];
          s[0] += a[k][j];
          s[1] = fmaf(a[k][j], e.xh[j], s[1]);
          s[2] += v[k][j];
          s[3] = fmaf(v[k][j], e.xh[j], s[3]);
        }
      }
    }
    RowSums<256, CURVED ? 2 : 4>::run(s, sm, turn);
    if constexpr (!CURVED) {
      const float count = (float)(p.cols - c0 < CHUNK ? p.cols - c0 : CHUNK), am = s[0] / count, vmean = s[2] / count;
      float t[1] = {0.f};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int n = (int)(p.cols - c0) - (threadIdx.x + k * 256) * 8;
#pragma unroll
        for (int j = 0; j < 8; ++j) t[0] = fmaf(j < n ? v[k][j] - vmean : 0.f, a[k][j] - am, t[0]);
      }
      RowSums<256, 1>::run(t, sm2, turn2);
      if (threadIdx.x == 0) p.chunk[item * K + 4] = t[0];
    }
    if (threadIdx.x == 0)
#pragma unroll
      for (int i = 0; i < (CURVED ? 2 : 4); ++i) p.chunk[item * K + i] = s[i];
  }
}

// 2 (ln_join for the sums of q gamma): sums of a row's chunks, joined by a wave; the last one = those around the chunks' means +
// the means' own spread.
__global__ __launch_bounds__(256) void ln_bwd2_join(LnArgs p, long chunks) {
  const int lane = threadIdx.x & 63;
  const float cols = (float)p.cols, last = (float)(p.cols - (chunks - 1) * CHUNK);
  for (long row = (long)blockIdx.x * 4 + (threadIdx.x >> 6); row < p.rows; row += (long)gridDim.x * 4) {
    const float* part = p.chunk + row * chunks * 5;
    float s[4] = {};
    for (long i = lane; i < chunks; i += 64)
#pragma unroll
      for (int k = 0; k < 4; ++k) s[k] += part[i * 5 + k];
#pragma unroll
    for (int k = 0; k < 4; ++k) s[k] = lanes_sum<64>(s[k]);
    const float am = s[0] / cols, vm = s[2] / cols;
    float t = 0.f;
    for (long i = lane; i < chunks; i += 64) {
      const float n = i + 1 < chunks ? (float)CHUNK : last;
      t += fmaf((part[i * 5 + 2] / n - vm) * n, part[i * 5] / n - am, part[i * 5 + 4]);
    }
    t = lanes_sum<64>(t);
    if (lane == 0) {
      float* out = p.row + row * ROW_SUMS;
#pragma unroll
      for (int k = 0; k < 4; ++k) out[k] = s[k];
      out[4] = t;
    }
  }
}

// 3: both cotangents and the affine sums of a row group.
template <typename T, int EPI>
__global__ __launch_bounds__(256) void ln_bwd2_stream(LnArgs p) {
  if (EPI) drop_state(p.drop);
  const int c = (int)((blockIdx.x * 256u + threadIdx.x) * 8), cols = (int)p.cols, n = cols - c;
  if (n <= 0) return;
  const float inv = 1.f / (float)cols;
  const bool curved = EPI == 2 && p.act > 1.f;
  float ga[8], be[8], dg[8], db[8];
  load_param<T>(p.gamma, p.param_f32, c, n, 1.f, ga);
  if (EPI == 2) load_param<T>(p.beta, p.param_f32, c, n, 0.f, be);
#pragma unroll
  for (int j = 0; j < 8; ++j) dg[j] = db[j] = 0.f;
  for (long row = blockIdx.y; row < p.rows; row += gridDim.y) {
    Eight<EPI, true> e;
    float v[8], gg[8], gx[8];
    load8((const T*)p.x + row * p.ld_x + c, n, e.xh);
    load8((const T*)p.gy + row * p.ld_gy + c, n, e.g);
    load8((const T*)p.ggx + row * p.ld_ggx + c, n, v);
    const float mean = p.mean[row], rstd = p.rstd[row];
    const float* rs = p.row + row * ROW_SUMS;
    const float am = rs[0] * inv, ax = rs[1] * inv, vm = rs[2] * inv, vx = rs[3] * inv;
    const float sv = rs[4] * inv - vx * ax;
    const float q0 = curved ? rs[5] * inv : 0.f, q1 = curved ? rs[6] * inv : 0.f;
    const float c0 = -rstd * q0, c1 = -rstd * ax, c2 = -rstd * rstd * vx;
    const float c3 = -rstd * (q1 + rstd * (sv - vx * ax));
    e.make(p, row, c, mean, rstd, ga, be);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float t = rstd * (v[j] - vm - e.xh[j] * vx);
      const float q = EPI == 2 ? e.g[j] * e.d2[j] * ga[j] * t : 0.f, g1 = EPI == 2 ? e.g[j] * e.d1[j] : e.g[j];
      gg[j] = (EPI == 2 ? e.d1[j] * ga[j] : ga[j]) * t;
      gx[j] = fmaf(t, c1, fmaf(fmaf(g1, ga[j], -am), c2, fmaf(e.xh[j], c3, c0)));
      dg[j] = fmaf(g1, t, dg[j]);
      if (EPI == 2) {
        gx[j] = fmaf(q * ga[j], rstd, gx[j]);
        dg[j] = fmaf(q, e.xh[j], dg[j]);
        db[j] += q;
      }
    }
    if (EPI && p.drop.t) drop_apply(p.drop, e.w, gg);
    store8((T*)p.ggy + row * p.ld_ggy + c, n, gg);
    store8((T*)p.out + row * p.ld_out + c, n, gx);
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
  const unsigned items = ln_items(a.rows, a.cols);
  ln_bwd2_chunks<T, EPI, false><<<items, 256, 0, st>>>(a, chunks);
  ln_bwd2_join<<<ln_join_grid(a.rows), 256, 0, st>>>(a, chunks);
  if (EPI == 2 && a.act > 1.f) {
    ln_bwd2_chunks<T, EPI, true><<<items, 256, 0, st>>>(a, chunks);
    ln_join<2><<<ln_join_grid(a.rows), 256, 0, st>>>(a.chunk, a.rows, chunks, a.row, 5);
  }
  ln_bwd2_stream<T, EPI><<<ln_stream_grid(a.rows, a.cols), 256, 0, st>>>(a);
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
    if (a.act != 1.f) ln_bwd2_rows<T, G, NV, 2><<<groups, G > 64 ? G : 256, 0, st>>>(a);                     \
    else if (a.drop.t) ln_bwd2_rows<T, G, NV, 1><<<groups, G > 64 ? G : 256, 0, st>>>(a);                    \
    else ln_bwd2_rows<T, G, NV, 0><<<groups, G > 64 ? G : 256, 0, st>>>(a);                                  \
  }
  LN_BWD_SHAPES(SHAPE)
#undef SHAPE
}

}  // namespace

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
  FCD_REQUIRE(d->rows == 0 || (mean && rstd), "%s: mean / rstd are NULL", who);
  FCD_TRY(ln_check_scratch(who, d, FCD_LN_BWD2, dgamma, dbeta, workspace, workspace_bytes, &a));
  const int64_t ps = fcd_dt_bytes(d->param_dtype) * d->cols, ss = 4 * d->rows;
  const Bytes written[] = {{"dgamma", dgamma, ps}, {"dbeta", dbeta, ps}, {"workspace", workspace, (int64_t)workspace_bytes}};
  const Bytes read[] = {{"mean", mean, ss}, {"rstd", rstd, ss}, {"gamma", gamma, ps}, {"beta", beta, ps}, {"rng", d->rng, 16}};
  const RowView rows[] = {in[0], in[1], in[2], out[0], out[1]};
  FCD_TRY(ln_check_apart(who, d, written, 3, read, 5, rows, 5));
  for (const Bytes& b : read)
    for (const RowView& v : out) FCD_TRY(fcd_check_apart(who, b, v, d->rows, d->cols, es));
  a.x = x, a.gy = gy, a.ggx = ggx, a.gamma = gamma, a.beta = beta, a.out = gx, a.ggy = ggy;
  a.mean = (float*)mean, a.rstd = (float*)rstd;
  const int groups = ln_groups(d->rows, d->cols);
  hipStream_t st = fcd_stream(stream);
  if (d->rows) {
    if (d->dtype == FCD_DT_F32) launch<float>(a, groups, st);
    else if (d->dtype == FCD_DT_BF16) launch<bf16_t>(a, groups, st);
    else launch<f16_t>(a, groups, st);
    FCD_TRY(fcd_check_launch(who));
  }
  return dgamma || dbeta ? ln_finish(who, d, a, groups, dgamma, dbeta, accumulate, st) : FCD_OK;
}
