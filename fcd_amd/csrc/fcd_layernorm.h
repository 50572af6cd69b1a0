// Shared by the layer norm's three directions (layernorm_fwd.hip, layernorm_bwd.hip, layernorm_bwd2.hip).
#pragma once
#include "fcd_rows.h"

struct LnArgs {
  const void *x, *res, *gy, *ggx, *gamma, *beta;
  void *out, *ggy;
  float *mean, *rstd;      // written by fwd, read by bwd / bwd2
  float* partial;          // scratch, [groups][2][cols]: a workgroup's sums of dgamma and dbeta; or NULL
  float *chunk, *row;      // scratch of rows that are split: [rows][chunks][K] sums and [rows][ROW_SUMS] joined ones
  long rows, cols, ld_x, ld_res, ld_gy, ld_ggx, ld_out, ld_ggy;
  float eps, act;
  int param_f32;
  Drop drop;
};

// layernorm.hip
int ln_check(const char* who, const FcdLayerNormDesc* d, LnArgs* a);
int ln_check_vectors(const char* who, const FcdLayerNormDesc* d, const void* gamma, const void* beta, const void* mean,
                     const void* rstd);
int ln_check_scratch(const char* who, const FcdLayerNormDesc* d, int pass, const void* dgamma, const void* dbeta, void* workspace,
                     size_t workspace_bytes, LnArgs* a);
// the written vectors w[nw] share memory with nothing: not with one another, the read ones r[nr] or the row tensors t[nt]
int ln_check_apart(const char* who, const FcdLayerNormDesc* d, const Bytes* w, int nw, const Bytes* r, int nr, const RowView* t,
                   int nt);
int ln_finish(const char* who, const FcdLayerNormDesc* d, const LnArgs& a, int groups, void* dgamma, void* dbeta, int accumulate,
              hipStream_t st);
int ln_groups(int64_t rows, int64_t cols);   // workgroups (row groups of split rows) of the backward passes
bool ln_few_rows(int64_t rows, int64_t cols);   // the first backward pass sums its columns apart from the rows (ln_bwd_few)

// Where a row lives: G threads with NV units of 8 elements each.  G <= 64: the row's sums stay inside a wave, and a workgroup
// of 256 works on 256 / G rows with no barrier; G > 64: one workgroup per row, one barrier per sum.  The forward pass keeps
// two units a thread (fewer waves meet at the barrier); the backward passes hold the affine sums as well and keep one.
// Longer rows than the last shape takes are split (below).
#define LN_FWD_SHAPES(F) \
  F(4, 1) F(8, 1) F(16, 1) F(32, 1) F(64, 1) F(64, 2) F(256, 1) F(256, 2) F(512, 2) F(1024, 2)
#define LN_BWD_SHAPES(F) \
  F(4, 1) F(8, 1) F(16, 1) F(32, 1) F(64, 1) F(128, 1) F(256, 1) F(512, 1) F(1024, 1)

struct LnShape {
  int g, nv;   // g 0: split rows
};

static inline LnShape ln_bwd_shape(int64_t cols) {
  const int64_t units = (cols + 7) / 8;
#define PICK(G, NV) \
  if (units <= (G) * (NV)) return {G, NV};
  LN_BWD_SHAPES(PICK)
#undef PICK
  return {0, 0};
}
constexpr int64_t LN_FWD_MAX = 16384;   // the last forward shape's columns
static_assert(LN_FWD_MAX >= FCD_LN_WHOLE, "");

// Split rows: one kernel sums chunks of a row, one joins the chunks of every row, and one streams: its workgroups own 2048
// columns, keep their parameters and affine sums in registers and walk down a group of rows whose sums are known, with no
// barrier.  The operands are read once more than by the shapes above, which is what a row of any length and a few long rows
// (one workgroup each would leave the card idle) cost.
constexpr int CHUNK = 8192;             // columns of a chunk: 256 threads, 4 units each
constexpr int ROW_SUMS = 7;
static inline int64_t ln_chunks(int64_t cols) { return (cols + CHUNK - 1) / CHUNK; }
static inline unsigned ln_items(int64_t rows, int64_t cols) {
  const __int128 n = (__int128)rows * ln_chunks(cols);
  return (unsigned)(n < 16384 ? n : 16384);
}
static inline dim3 ln_stream_grid(int64_t rows, int64_t cols) { return dim3((unsigned)((cols + 2047) / 2048), ln_groups(rows, cols)); }
static inline unsigned ln_join_grid(int64_t rows) { return (unsigned)(rows < 65536 ? (rows + 3) / 4 : 16384); }

// The row of a thread (wave-uniform where it can be, so that row addresses live in scalar registers) and its first column.
template <int G, int TH>
__device__ __forceinline__ long first_row() {
  if constexpr (G == TH) return blockIdx.x;
  if constexpr (G == 64) return (long)blockIdx.x * (TH / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  return (long)blockIdx.x * (TH / G) + threadIdx.x / G;
}

template <typename T, typename N>
__device__ __forceinline__ void load_param(const void* p, int f32, N c, N n, float none, float (&v)[8]) {
  if (!p) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = none;
  } else if (f32) {
    load8((const float*)p + c, n, v);
  } else {
    load8((const T*)p + c, n, v);
  }
}

// A lane's unit of a row, prefetched: its 8 elements, or at a ragged end the row's last 8, which settle() moves down when they
// are used.  (Lane by lane loads of an end would have to be waited for where they are issued.)  G = 4 may meet rows of less
// than 8, whose elements are loaded one by one.
template <typename T, int G>
__device__ __forceinline__ void fetch8(const T* row, int c, int cols, typename Oct<T>::type& o) {
  if (G == 4 && cols < 8) {
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = j < cols - c ? row[c + j] : (T)0.f;
  } else {
    o = *reinterpret_cast<const typename Oct<T>::type*>(row + (c < cols - 8 ? c : cols - 8));
  }
}

// n: how many of the 8 exist (0 or less: none, all zero)
template <typename T, int G>
__device__ __forceinline__ void settle(typename Oct<T>::type& o, int cols, int n) {
  if (n < 8 && !(G == 4 && cols < 8 && n > 0)) {
    const typename Oct<T>::type z = {};
    const int d = 8 - n;
    typename Oct<T>::type r = d & 4 ? __builtin_shufflevector(o, z, 4, 5, 6, 7, 8, 8, 8, 8) : o;
    r = d & 2 ? __builtin_shufflevector(r, z, 2, 3, 4, 5, 6, 7, 8, 8) : r;
    r = d & 1 ? __builtin_shufflevector(r, z, 1, 2, 3, 4, 5, 6, 7, 8) : r;
    o = n > 0 ? r : z;
  }
}

template <typename T>
__device__ __forceinline__ void widen(const typename Oct<T>::type& o, float (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = (float)o[j];
}

// Waits here for the load into `o`.  Loads and stores retire in one order, and whether a store was issued depends on the lane:
// a wait for a prefetch that stands behind a row's stores is a wait for the stores as well.  So the next row's loads are
// waited for in front of them.
template <typename T>
__device__ __forceinline__ void arrive(typename Oct<T>::type& o) {
  typedef int Quad __attribute__((ext_vector_type(4)));
  struct Quads { Quad q[sizeof(T) / 2]; };
  Quads t = __builtin_bit_cast(Quads, o);
#pragma unroll
  for (unsigned i = 0; i < sizeof(T) / 2; ++i) asm volatile("" : "+v"(t.q[i]));
  o = __builtin_bit_cast(typename Oct<T>::type, t);
}

// ---------------------------------------------------------------- sums -----------------
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}

// a + b after the exchange of a's upper half with b's lower half: sums of a's halves in the lower 32 lanes, of b's in the upper.
__device__ __forceinline__ float swap32_add(float a, float b) {
  const auto s = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b), false, false);
  const unsigned lo = s[0], hi = s[1];
  return __builtin_bit_cast(float, lo) + __builtin_bit_cast(float, hi);
}

// The same between odd rows of a and even rows of b (16 lanes each): rows 0 and 2 get sums of a's rows, 1 and 3 of b's.
__device__ __forceinline__ float swap16_add(float a, float b) {
  const auto s = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b), false, false);
  const unsigned lo = s[0], hi = s[1];
  return __builtin_bit_cast(float, lo) + __builtin_bit_cast(float, hi);
}

// Sum over groups of G neighbouring lanes, in every lane: swaps inside quads, mirrors of 8 and 16 lanes (all lanes of a
// smaller group already hold the same value there), then the row and half swaps of gfx950.  No LDS round trip.
template <int G>
__device__ __forceinline__ float lanes_sum(float v) {
  if constexpr (G >= 2) v += dpp<0xB1>(v);
  if constexpr (G >= 4) v += dpp<0x4E>(v);
  if constexpr (G >= 8) v += dpp<0x141>(v);
  if constexpr (G >= 16) v += dpp<0x140>(v);
  if constexpr (G >= 32) v = swap16_add(v, v);
  if constexpr (G >= 64) v = swap32_add(v, v);
  return v;
}

__device__ __forceinline__ float lane_value(float v, int lane) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}

// Sums of K values over the G threads of a row, in every thread (from a wave on in scalar registers).  A wave's sums share
// their exchanges: each swap folds two of them at once, so that four cost little more than one, and end up in the lanes home(k).
// More than a wave: one barrier; `turn` alternates between two buffers, and a wave writes to one again only behind the barrier of
// the other, which every wave reaches after its reads.
template <int G, int K>
struct RowSums {
  static_assert(K >= 1 && K <= 4, "");
  static constexpr int WAVES = G > 64 ? G / 64 : 1;
  __device__ __forceinline__ static constexpr int home(int k) { return 32 * (k & 1) + 8 * (k & 2); }

  __device__ __forceinline__ static float fold(const float (&s)[K]) {
    if constexpr (K == 1) return lanes_sum<64>(s[0]);
    if constexpr (K == 2) {
      const float r = swap32_add(s[0], s[1]);
      return lanes_sum<16>(swap16_add(r, r));
    }
    if constexpr (K > 2) return lanes_sum<16>(swap16_add(swap32_add(s[0], s[1]), swap32_add(s[2], s[K - 1])));
  }

  __device__ __forceinline__ static void run(float (&s)[K], float* sm, int& turn) {
    if constexpr (G < 64) {
#pragma unroll
      for (int k = 0; k < K; ++k) s[k] = lanes_sum<G>(s[k]);
    } else {
      const float r = fold(s);
      if constexpr (G == 64) {
#pragma unroll
        for (int k = 0; k < K; ++k) s[k] = lane_value(r, home(k));
      } else {
        float* buf = sm + turn * WAVES * K;
        turn ^= 1;
        const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
        int mine = -1;
#pragma unroll
        for (int k = 0; k < K; ++k) mine = lane == home(k) ? k : mine;
        if (mine >= 0) buf[mine * WAVES + w] = r;
        __syncthreads();
        // sum k's waves in WAVES neighbouring lanes
        static_assert(K * WAVES <= 64, "");
        const float a = lanes_sum<WAVES>(buf[lane < K * WAVES ? lane : 0]);
#pragma unroll
        for (int k = 0; k < K; ++k) s[k] = lane_value(a, k * WAVES);
      }
    }
  }
};

// A wave without elements (a row of 1536 has 192 units for 256 threads): its part in a row's sums is their barriers and a
// zero.  It leaves the rest of the row loop out, to the gain of the other waves on its SIMD.
template <int G>
__device__ __forceinline__ bool idle_wave(int cols) {
  return G > 64 && __builtin_amdgcn_readfirstlane(threadIdx.x & ~63u) * 8 >= cols;
}

template <int G, int K>
__device__ __forceinline__ void idle_sums(float* sm, int& turn) {
  float s[K] = {};
  RowSums<G, K>::run(s, sm, turn);
}

// ---------------------------------------------------------------- activations ----------
// The smooth ones from one hardware exponential and one hardware reciprocal (a step of fp32 each).  exp(u) as 2^(u log2 e)
// loses |u| / 2 steps relative; what it is used in changes by at most |u| s (1 - s) < 0.23 times that.
// mish, e = exp(u), n = e (e + 2): tanh(log(1 + e)) = n / (n + 2), its derivative w = 4 e (1 + e) / (n + 2)^2.  Beyond u = 20
// that is 1 in fp32 and w below 2e-17, where u itself may be anything: e and the factor of w take u clamped (NaN stays NaN).
__device__ __forceinline__ float fast_exp(float u) { return __builtin_amdgcn_exp2f(u * 1.44269504088896341f); }

// The activation (d0) of 8 values, or its first (d1) and second (d2) derivative; what is NULL is not computed.
__device__ __forceinline__ void ln_act8(const float (&u)[8], float code, float* d0, float* d1, float* d2) {
  if (code == FCD_ACT_SILU) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float sg = __builtin_amdgcn_rcpf(1.f + fast_exp(-u[j])), ns = 1.f - sg;
      if (d0) d0[j] = u[j] * sg;
      if (d1) d1[j] = fmaf(u[j] * sg, ns, sg);
      if (d2) d2[j] = sg * ns * fmaf(u[j], ns - sg, 2.f);
    }
  } else if (code == FCD_ACT_MISH) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float uc = u[j] > 20.f ? 20.f : u[j];
      const float e = fast_exp(uc), n = e * (e + 2.f), r = __builtin_amdgcn_rcpf(n + 2.f), th = n * r;
      if (d0) d0[j] = u[j] * th;
      const float w = 4.f * e * (1.f + e) * r * r;
      if (d1) d1[j] = fmaf(uc, w, th);
      if (d2) {
        const float sg = e * __builtin_amdgcn_rcpf(1.f + e);
        d2[j] = w * fmaf(uc, (1.f - sg) - 2.f * th * sg, 2.f);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float s = u[j] > 0.f ? 1.f : code;
      if (d0) d0[j] = u[j] * s;
      if (d1) d1[j] = s;
      if (d2) d2[j] = 0.f;
    }
  }
}

// ---------------------------------------------------------------- backward passes ------
// What the backward passes need of 8 elements of x and gy: xhat, drop(gy), and behind an activation act'(u), act''(u).
// Absent elements (gy 0) come out with drop(gy) = 0.
template <int EPI, bool SECOND>
struct Eight {
  float xh[8], g[8], d1[8], d2[8];
  uint32_t w[4];

  __device__ __forceinline__ void make(const LnArgs& p, long row, int c, float mean, float rstd, const float (&ga)[8],
                                       const float (&be)[8]) {
    if (EPI && p.drop.t) {
      drop_draw8(p.drop, (uint64_t)(row * p.cols + c), w);
      drop_apply(p.drop, w, g);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) xh[j] = (xh[j] - mean) * rstd;
    if (EPI == 2) {
      float u[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) u[j] = fmaf(xh[j], ga[j], be[j]);
      ln_act8(u, p.act, nullptr, d1, SECOND ? d2 : nullptr);
    }
  }
};

// Affine sums of a workgroup whose threads each kept NV * 8 columns in registers: over the groups of a wave by exchanges, over
// the waves through LDS, in a fixed order; then to the workgroup's place in the scratch.
template <int G, int NV>
constexpr int affine_lds() { return G > 64 ? 1 : 4 * 2 * G * NV * 8; }

template <int G, int NV>
__device__ __forceinline__ void write_partial(const LnArgs& p, float (&dg)[NV][8], float (&db)[NV][8], float* sm) {
  float* part = p.partial + (long)blockIdx.x * 2 * p.cols;
  const int lane = threadIdx.x % G, cols = (int)p.cols;
  if constexpr (G > 64) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (lane + k * G) * 8;
      store8(part + c, cols - c, dg[k]);
      store8(part + cols + c, cols - c, db[k]);
    }
  } else {
    const int w = threadIdx.x >> 6;
    constexpr int W = G * NV * 8;
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float a = dg[k][j], b = db[k][j];
#pragma unroll
        for (int o = G; o < 64; o <<= 1) {
          a += __shfl_xor(a, o, 64);
          b += __shfl_xor(b, o, 64);
        }
        if ((threadIdx.x & 63) < G) {
          sm[(w * 2 + 0) * W + (lane + k * G) * 8 + j] = a;
          sm[(w * 2 + 1) * W + (lane + k * G) * 8 + j] = b;
        }
      }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * W; i += 256) {
      const int which = i / W, c = i % W;
      if (c < cols) part[which * cols + c] = (sm[i] + sm[2 * W + i]) + (sm[4 * W + i] + sm[6 * W + i]);
    }
  }
}

// Sums of a row's chunks, joined by a wave.
template <int K>
__global__ __launch_bounds__(256) void ln_join(const float* chunk, long rows, long chunks, float* row_sums, int first) {
  const int lane = threadIdx.x & 63;
  for (long row = (long)blockIdx.x * 4 + (threadIdx.x >> 6); row < rows; row += (long)gridDim.x * 4) {
    float s[K];
#pragma unroll
    for (int k = 0; k < K; ++k) s[k] = 0.f;
    for (long i = lane; i < chunks; i += 64)
#pragma unroll
      for (int k = 0; k < K; ++k) s[k] += chunk[(row * chunks + i) * K + k];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      s[k] = lanes_sum<64>(s[k]);
      if (lane == 0) row_sums[row * ROW_SUMS + first + k] = s[k];
    }
  }
}
