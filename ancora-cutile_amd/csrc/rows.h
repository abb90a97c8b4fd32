// Rows of fp32 or bf16 values in pieces of VEC elements, widened to fp32 in registers: what the operators that are
// indexed by token (embed_rows.hip, dispatch.hip) read and write.
#pragma once
#include "common.h"

namespace anc_rows {

// One rounding to nearest even; NaN stays NaN (the integer formula of anc_bf16_rne_bits carries some NaN into zero).
__device__ __forceinline__ uint32_t bf16_bits(float x) {
  return (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)x);
}
__device__ __forceinline__ uint32_t bf16_pair(float a, float b) { return bf16_bits(a) | (bf16_bits(b) << 16); }

template <int T> struct Elem;
template <> struct Elem<ANC_F32> { using type = float; };
template <> struct Elem<ANC_BF16> { using type = uint16_t; };
template <int T> using elem_t = typename Elem<T>::type;

// VEC elements at p, in registers as they lie in memory: loads first, widening where the values are needed.
template <int T, int VEC> struct Raw;
template <> struct Raw<ANC_BF16, 8> { anc_u32x4 q; };
template <> struct Raw<ANC_BF16, 4> { anc_u32x2 q; };
template <> struct Raw<ANC_BF16, 2> { uint32_t q; };
template <> struct Raw<ANC_BF16, 1> { uint16_t q; };
template <> struct Raw<ANC_F32, 8> { anc_f32x4 a, b; };      // (sums of bf16 rows)
template <> struct Raw<ANC_F32, 4> { anc_f32x4 a; };
template <> struct Raw<ANC_F32, 2> { anc_f32x2 a; };
template <> struct Raw<ANC_F32, 1> { float a; };

template <int T, int VEC> __device__ __forceinline__ Raw<T, VEC> load(const elem_t<T> *p) {
  return *(const Raw<T, VEC> *)p;
}
template <int T, int VEC> __device__ __forceinline__ void widen(const Raw<T, VEC> &r, float (&x)[VEC]) {
  if constexpr (T == ANC_BF16 && VEC == 8) {
    const uint32_t w[4] = {r.q.x, r.q.y, r.q.z, r.q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  } else if constexpr (T == ANC_BF16 && VEC == 4) {
    x[0] = __uint_as_float(r.q.x << 16);
    x[1] = __uint_as_float(r.q.x & 0xFFFF0000u);
    x[2] = __uint_as_float(r.q.y << 16);
    x[3] = __uint_as_float(r.q.y & 0xFFFF0000u);
  } else if constexpr (T == ANC_BF16 && VEC == 2) {
    x[0] = __uint_as_float(r.q << 16);
    x[1] = __uint_as_float(r.q & 0xFFFF0000u);
  } else if constexpr (T == ANC_BF16) {
    x[0] = __uint_as_float((uint32_t)r.q << 16);
  } else if constexpr (VEC == 8) {
    x[0] = r.a.x; x[1] = r.a.y; x[2] = r.a.z; x[3] = r.a.w;
    x[4] = r.b.x; x[5] = r.b.y; x[6] = r.b.z; x[7] = r.b.w;
  } else if constexpr (VEC == 4) {
    x[0] = r.a.x; x[1] = r.a.y; x[2] = r.a.z; x[3] = r.a.w;
  } else if constexpr (VEC == 2) {
    x[0] = r.a.x; x[1] = r.a.y;
  } else {
    x[0] = r.a;
  }
}
template <int T, int VEC> __device__ __forceinline__ Raw<T, VEC> narrow(const float (&x)[VEC]) {
  Raw<T, VEC> r;
  if constexpr (T == ANC_BF16 && VEC == 8) {
    r.q = anc_u32x4{bf16_pair(x[0], x[1]), bf16_pair(x[2], x[3]), bf16_pair(x[4], x[5]), bf16_pair(x[6], x[7])};
  } else if constexpr (T == ANC_BF16 && VEC == 4) {
    r.q = anc_u32x2{bf16_pair(x[0], x[1]), bf16_pair(x[2], x[3])};
  } else if constexpr (T == ANC_BF16 && VEC == 2) {
    r.q = bf16_pair(x[0], x[1]);
  } else if constexpr (T == ANC_BF16) {
    r.q = (uint16_t)bf16_bits(x[0]);
  } else if constexpr (VEC == 8) {
    r.a = anc_f32x4{x[0], x[1], x[2], x[3]};
    r.b = anc_f32x4{x[4], x[5], x[6], x[7]};
  } else if constexpr (VEC == 4) {
    r.a = anc_f32x4{x[0], x[1], x[2], x[3]};
  } else if constexpr (VEC == 2) {
    r.a = anc_f32x2{x[0], x[1]};
  } else {
    r.a = x[0];
  }
  return r;
}
// ONCE: past the caches, for rows so large that whoever reads them next does not find them there anyway (see kCached).
template <int T, int VEC, bool ONCE> __device__ __forceinline__ Raw<T, VEC> load(const elem_t<T> *p) {
  Raw<T, VEC> r;
  if constexpr (!ONCE) {
    r = *(const Raw<T, VEC> *)p;
  } else if constexpr (T == ANC_BF16) {
    r.q = anc_ld_stream((const decltype(r.q) *)p);
  } else {
    r.a = anc_ld_stream((const decltype(r.a) *)p);
    if constexpr (VEC == 8) r.b = anc_ld_stream((const anc_f32x4 *)p + 1);
  }
  return r;
}
template <int T, int VEC, bool ONCE> __device__ __forceinline__ void store(elem_t<T> *p, const Raw<T, VEC> &r) {
  if constexpr (!ONCE) {
    *(Raw<T, VEC> *)p = r;
  } else if constexpr (T == ANC_BF16) {
    anc_st_stream((decltype(Raw<T, VEC>::q) *)p, r.q);
  } else {
    anc_st_stream((decltype(Raw<T, VEC>::a) *)p, r.a);
    if constexpr (VEC == 8) anc_st_stream((anc_f32x4 *)p + 1, r.b);
  }
}
template <int T, int VEC, bool ONCE> __device__ __forceinline__ void store(elem_t<T> *p, const float (&x)[VEC]) {
  store<T, VEC, ONCE>(p, narrow<T, VEC>(x));
}
template <int T, int VEC> __device__ __forceinline__ void store(elem_t<T> *p, const Raw<T, VEC> &r) { *(Raw<T, VEC> *)p = r; }
template <int T, int VEC> __device__ __forceinline__ void store(elem_t<T> *p, const float (&x)[VEC]) {
  *(Raw<T, VEC> *)p = narrow<T, VEC>(x);
}

// i / d for i < 2^31 as one multiplication (64-bit division by a value that is not known to the compiler is some hundred instructions):
// m = ceil(2^(31 + s) / d) with 2^s >= d is below 2^32 + 1 and m i / 2^(31 + s) exceeds i / d by less than 1 / d.
struct FastDiv {
  uint32_t d, mul;
  int shift;
  __device__ __forceinline__ uint32_t div(uint32_t i) const { return d == 1 ? i : __umulhi(i, mul) >> shift; }
};
inline FastDiv fast_div(uint32_t d) {
  FastDiv f{d, 0, 0};
  if (d == 1) return f;
  int s = 0;
  while ((1ull << s) < d) ++s;                       // 2^s >= d >= 2, s >= 1
  f.mul = (uint32_t)(((1ull << (31 + s)) + d - 1) / d);
  f.shift = s - 1;
  return f;
}

// ---- host side: which piece a call's rows allow
constexpr int64_t kMostPieces = (1ll << 31) - 1;     // of one launch (FastDiv)
// Bytes up to which rows go through the caches. A lookup of 16 MiB and a copy of it afterwards: 12.6 us, with its stores past the caches 14.7;
// one of 199 MB: 149 us, past the caches 145, and the lookup alone 72 and 66.
constexpr int64_t kCached = 64ll << 20;
struct Ptr { uint64_t p; int type; };
inline int64_t elem_size(int type) { return type == ANC_F32 ? 4 : 2; }
inline bool type_ok(int type) { return type == ANC_F32 || type == ANC_BF16; }
// 16 bytes of the widest type where every row starts so aligned (a lane's neighbour then reads the next 16 bytes): 8 elements of bf16 rows, 4
// where fp32 rows take part; else pairs where H is even and the pointers allow them, else single elements.
template <int N> inline int piece(int64_t H, const Ptr (&ps)[N]) {
  int wide = 8;
  for (const Ptr &q : ps)
    if (q.type == ANC_F32) wide = 4;
  bool wides = H % wide == 0, by2 = H % 2 == 0;
  for (const Ptr &q : ps) {
    wides = wides && q.p % (uint64_t)(wide * elem_size(q.type)) == 0;
    by2 = by2 && q.p % (uint64_t)(2 * elem_size(q.type)) == 0;
  }
  return wides ? wide : by2 ? 2 : 1;
}
template <int V> struct Int { static constexpr int value = V; };
template <typename F> inline void with_type(int type, F &&f) {
  if (type == ANC_F32) f(Int<ANC_F32>{}); else f(Int<ANC_BF16>{});
}
template <typename F> inline void with_piece(int vec, F &&f) {
  if (vec == 8) f(Int<8>{}); else if (vec == 4) f(Int<4>{}); else if (vec == 2) f(Int<2>{}); else f(Int<1>{});
}

}  // namespace anc_rows
