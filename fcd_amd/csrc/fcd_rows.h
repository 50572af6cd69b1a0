// Shared by layernorm.hip and dropout.hip: element types, 8-element accesses at any alignment, the dropout generator, and the
// host checks of row tensors.
#pragma once
#include "fcd_common.h"

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

// A lane's unit of work is 8 consecutive elements: one 16-byte access of a 16-bit type, two of fp32, and exactly one
// generator block of dropout.  Global accesses of gfx950 take any alignment, so rows of odd length need no other path.
template <typename T> struct Oct;
template <> struct Oct<float> { typedef float type __attribute__((ext_vector_type(8), aligned(4))); };
template <> struct Oct<bf16_t> { typedef bf16_t type __attribute__((ext_vector_type(8), aligned(2))); };
template <> struct Oct<f16_t> { typedef f16_t type __attribute__((ext_vector_type(8), aligned(2))); };

// n: how many of the 8 exist; the others read as 0 and are not written
template <typename T, typename N>
__device__ __forceinline__ void load8(const T* p, N n, float (&v)[8]) {
  if (n >= 8) {
    const typename Oct<T>::type o = *reinterpret_cast<const typename Oct<T>::type*>(p);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (float)o[j];
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < n ? (float)p[j] : 0.f;
  }
}

template <typename T, typename N>
__device__ __forceinline__ void store8(T* p, N n, const float (&v)[8]) {
  if (n >= 8) {
    typename Oct<T>::type o;
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = (T)v[j];
    *reinterpret_cast<typename Oct<T>::type*>(p) = o;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) p[j] = (T)v[j];
  }
}

// ---------------------------------------------------------------- dropout --------------
struct Drop {
  uint64_t seed, offset;
  const uint64_t* rng;   // device words {seed, offset} in place of seed, added to offset; or NULL
  float scale;           // 65536 / (65536 - t); 0 if everything is dropped
  uint32_t t;            // dropped where the 16 bits are below t; 0: no dropout
  uint32_t below;        // (t << 16) - 1
};

__device__ __forceinline__ uint32_t xor3(uint32_t a, uint32_t b, uint32_t c) { return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96); }

// seed and first block, read once per thread
__device__ __forceinline__ void drop_state(Drop& d) {
  if (d.t && d.rng) {
    d.seed = d.rng[0];
    d.offset += d.rng[1];
  }
}

// One block of Philox4x32-10.  (A product's two halves come from one 32 x 32 -> 64 bit multiply-add; three-way xors are
// single instructions of gfx950.)
__device__ __forceinline__ void drop_block(const Drop& d, uint64_t block, uint32_t (&w)[4]) {
  uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = 0, c3 = 0;
  uint32_t k0 = (uint32_t)d.seed, k1 = (uint32_t)(d.seed >> 32);
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t p0 = (uint64_t)0xD2511F53u * c0, p1 = (uint64_t)0xCD9E8D57u * c2;
    c0 = xor3((uint32_t)(p1 >> 32), c1, k0);
    c1 = (uint32_t)p1;
    c2 = xor3((uint32_t)(p0 >> 32), c3, k1);
    c3 = (uint32_t)p0;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  w[0] = c0, w[1] = c1, w[2] = c2, w[3] = c3;
}

// The eight 16-bit draws of the elements i ... i + 7 of the matrix: one block if i is a multiple of 8, else the end of one and
// the beginning of the next.
__device__ __forceinline__ void drop_draw8(const Drop& d, uint64_t i, uint32_t (&w)[4]) {
  const uint64_t block = d.offset + (i >> 3);
  const uint32_t phase = (uint32_t)i & 7u;
  drop_block(d, block, w);
  if (phase) {
    asm volatile("");                    // (a branch: without it the compiler draws both blocks always and selects)
    uint32_t n[4];
    drop_block(d, block + 1, n);
    // the two blocks as eight words, moved down by `phase` halves (scalars: an array would be indexed in memory)
    const bool m4 = phase & 4u, m2 = phase & 2u, m1 = phase & 1u;
    uint32_t a0 = m4 ? w[2] : w[0], a1 = m4 ? w[3] : w[1], a2 = m4 ? n[0] : w[2], a3 = m4 ? n[1] : w[3];
    uint32_t a4 = m4 ? n[2] : n[0], a5 = m4 ? n[3] : n[1];
    a0 = m2 ? a1 : a0, a1 = m2 ? a2 : a1, a2 = m2 ? a3 : a2, a3 = m2 ? a4 : a3, a4 = m2 ? a5 : a4;
    w[0] = m1 ? a0 >> 16 | a1 << 16 : a0;
    w[1] = m1 ? a1 >> 16 | a2 << 16 : a1;
    w[2] = m1 ? a2 >> 16 | a3 << 16 : a2;
    w[3] = m1 ? a3 >> 16 | a4 << 16 : a3;
  }
}

// A draw stays where it is at least t.  Both halves are compared in the upper 16 bits of a word, with (t << 16) - 1.
__device__ __forceinline__ void drop_apply(const Drop& d, const uint32_t (&w)[4], float (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[2 * j] = w[j] << 16 > d.below ? v[2 * j] * d.scale : 0.f;
    v[2 * j + 1] = w[j] > d.below ? v[2 * j + 1] * d.scale : 0.f;
  }
}

// ---------------------------------------------------------------- host checks ----------
static inline int fcd_dt_bytes(int dt) { return dt == FCD_DT_F32 ? 4 : (dt == FCD_DT_BF16 || dt == FCD_DT_F16) ? 2 : 0; }

static inline int fcd_make_drop(const char* who, double p, uint64_t seed, uint64_t offset, const uint64_t* rng, Drop* out) {
  FCD_REQUIRE(p >= 0.0 && p <= 1.0, "%s: the dropout probability must be in [0, 1]", who);
  FCD_REQUIRE(((uintptr_t)rng & 7u) == 0, "%s: rng must be 8-byte aligned", who);
  out->t = (uint32_t)__builtin_rint(p * 65536.0);
  out->below = (uint32_t)(((uint64_t)out->t << 16) - 1);
  out->scale = out->t < 65536u ? (float)(65536.0 / (65536.0 - out->t)) : 0.f;
  out->seed = rng ? 0 : seed;
  out->offset = offset;
  out->rng = rng;
  return FCD_OK;
}

struct RowView {
  const char* name;
  const void* p;
  int64_t ld;
};

// A row tensor: present, aligned to its element, addressable, and (written) without rows that overlap.
static inline int fcd_check_rows(const char* who, const RowView& v, int64_t rows, int64_t cols, int esize, bool written) {
  FCD_REQUIRE(v.p || rows == 0 || cols == 0, "%s: %s is NULL", who, v.name);
  FCD_REQUIRE(((uintptr_t)v.p & (uintptr_t)(esize - 1)) == 0, "%s: %s is not aligned to its element type", who, v.name);
  FCD_REQUIRE(v.ld >= (written && rows > 1 ? cols : 0), "%s: row stride %lld of %s for %lld columns", who, (long long)v.ld,
              v.name, (long long)cols);
  FCD_REQUIRE(rows == 0 || (__int128)(rows - 1) * v.ld + cols < (__int128)1 << 58, "%s: %s is too large", who, v.name);
  return FCD_OK;
}

// An output and another tensor share memory without being the same tensor (column ranges of one wider tensor do not).
static inline int fcd_check_apart(const char* who, const RowView& out, const RowView& in, int64_t rows, int64_t cols, int esize,
                                  bool same_ok) {
  if (!out.p || !in.p || rows == 0 || cols == 0) return FCD_OK;
  const int64_t ld_o = rows > 1 ? out.ld : cols, ld_i = rows > 1 ? in.ld : cols;
  const __int128 a = (__int128)(uintptr_t)out.p, b = (__int128)(uintptr_t)in.p;
  const __int128 ea = a + ((__int128)(rows - 1) * ld_o + cols) * esize, eb = b + ((__int128)(rows - 1) * ld_i + cols) * esize;
  if (ea <= b || eb <= a) return FCD_OK;
  if (a == b && ld_o == ld_i && same_ok) return FCD_OK;
  if (ld_o == ld_i && ld_o > 0) {
    const __int128 diff = a > b ? a - b : b - a;
    const __int128 o = diff / esize % ld_o;
    if (diff % esize == 0 && o >= cols && o + cols <= ld_o) return FCD_OK;
  }
  fcd_set_error("%s: %s overlaps %s", who, out.name, in.name);
  return FCD_EINVAL;
}

// A vector or scratch that a call writes shares no byte with anything else of the call: workgroups run in any order.
struct Bytes {
  const char* name;
  const void* p;
  int64_t n;
};

static inline int fcd_check_apart(const char* who, const Bytes& a, const Bytes& b) {
  if (!a.p || !b.p || a.n <= 0 || b.n <= 0) return FCD_OK;
  const __int128 pa = (uintptr_t)a.p, pb = (uintptr_t)b.p;
  if (pa + a.n <= pb || pb + b.n <= pa) return FCD_OK;
  fcd_set_error("%s: %s overlaps %s", who, a.name, b.name);
  return FCD_EINVAL;
}

// ... with the elements of a row tensor (the gaps between its rows are free)
static inline int fcd_check_apart(const char* who, const Bytes& a, const RowView& v, int64_t rows, int64_t cols, int esize) {
  if (!a.p || !v.p || a.n <= 0 || rows <= 0 || cols <= 0) return FCD_OK;
  const __int128 lo = (__int128)(uintptr_t)a.p - (__int128)(uintptr_t)v.p, row = (__int128)cols * esize;
  const __int128 pitch = (__int128)(rows > 1 ? v.ld : 0) * esize;
  if (lo + a.n <= 0 || lo >= pitch * (rows - 1) + row) return FCD_OK;
  if (pitch > row && lo >= 0 && lo % pitch >= row && lo % pitch + a.n <= pitch) return FCD_OK;
  fcd_set_error("%s: %s overlaps %s", who, a.name, v.name);
  return FCD_EINVAL;
}

#define FCD_TRY(call)            \
  do {                           \
    const int rc_ = (call);      \
    if (rc_ != FCD_OK) return rc_; \
  } while (0)
