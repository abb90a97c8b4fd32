// Rows of fp32 or bf16 values in pieces of VEC elements, widened to fp32 in registers: what the operators that are
// indexed by token (embed_rows.hip, dispatch.hip) read and write.
//
// A piece is 16 bytes of the widest type at work (a lane's neighbour reads the next 16): 8 elements between bf16 rows, 4 where fp32 rows take
// part. Rows may start at any element: the accesses ask for the element's alignment only, which the hardware serves in one instruction.
// With TAIL (H no multiple of VEC) the last piece is the row's last VEC elements: it reads, and where that changes nothing also writes,
// elements of its neighbour once more. (Rows of 1001 bf16 values, a lookup of 16384: by single elements 27.9 us, so 14.3, rows of 1000 12.0.)
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
template <int A, int B> constexpr int piece_of = A == ANC_F32 || B == ANC_F32 ? 4 : 8;

// VEC elements in registers as they lie in memory: loads first, widening where the values are needed.
template <int T, int VEC> struct Raw;
template <> struct Raw<ANC_BF16, 8> { anc_u32x4 q; };
template <> struct Raw<ANC_BF16, 4> { anc_u32x2 q; };
template <> struct Raw<ANC_F32, 4> { anc_f32x4 q; };
template <> struct Raw<ANC_F32, 8> { anc_f32x4 q, r; };          // (sums of bf16 rows)
typedef anc_u32x4 u32x4_any __attribute__((aligned(2)));
typedef anc_u32x2 u32x2_any __attribute__((aligned(2)));
typedef anc_f32x4 f32x4_any __attribute__((aligned(4)));
template <int T, int VEC> struct Any;
template <> struct Any<ANC_BF16, 8> { using type = u32x4_any; };
template <> struct Any<ANC_BF16, 4> { using type = u32x2_any; };
template <int VEC> struct Any<ANC_F32, VEC> { using type = f32x4_any; };

// VEC elements of a row from `at` on, of which [first, last) are the piece's own and [0, last) there (last < VEC: the row is shorter than a piece).
struct Piece { int64_t at; int first, last; };
template <int VEC, bool TAIL> __device__ __forceinline__ Piece piece_at(int64_t col, int64_t H) {
  if (!TAIL || col + VEC <= H) return Piece{col, 0, VEC};
  if (H >= VEC) return Piece{H - VEC, (int)(VEC - (H - col)), VEC};
  return Piece{0, 0, (int)H};
}
// ONCE: past the caches, for rows so large that whoever reads them next does not find them there anyway (see kCached).
template <int T, int VEC, bool TAIL, bool ONCE = false>
__device__ __forceinline__ Raw<T, VEC> load(const elem_t<T> *row, const Piece &c) {
  using V = typename Any<T, VEC>::type;
  const elem_t<T> *p = row + c.at;
  Raw<T, VEC> r;
  if (!TAIL || c.last == VEC) {
    if constexpr (ONCE) r.q = __builtin_nontemporal_load((const V *)p);
    else r.q = *(const V *)p;
    if constexpr (T == ANC_F32 && VEC == 8) {
      if constexpr (ONCE) r.r = __builtin_nontemporal_load((const V *)p + 1);
      else r.r = *((const V *)p + 1);
    }
  } else {
    struct { elem_t<T> e[VEC]; } some;
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      some.e[k] = 0;
      if (k < c.last) some.e[k] = p[k];
    }
    r = __builtin_bit_cast(Raw<T, VEC>, some);
  }
  return r;
}
// OWN: the piece's own elements only, where a neighbour's must not be written twice (sums onto what is there).
template <int T, int VEC, bool TAIL, bool ONCE = false, bool OWN = false>
__device__ __forceinline__ void store(elem_t<T> *row, const Raw<T, VEC> &r, const Piece &c) {
  using V = typename Any<T, VEC>::type;
  elem_t<T> *p = row + c.at;
  if (!TAIL || (c.last == VEC && (!OWN || c.first == 0))) {
    if constexpr (ONCE) __builtin_nontemporal_store((V)r.q, (V *)p);
    else *(V *)p = r.q;
    if constexpr (T == ANC_F32 && VEC == 8) {
      if constexpr (ONCE) __builtin_nontemporal_store((V)r.r, (V *)p + 1);
      else *((V *)p + 1) = r.r;
    }
  } else {
    struct S { elem_t<T> e[VEC]; };
    const S some = __builtin_bit_cast(S, r);
#pragma unroll
    for (int k = 0; k < VEC; ++k)
      if (k >= c.first && k < c.last) p[k] = some.e[k];
  }
}
template <int T, int VEC> __device__ __forceinline__ void widen(const Raw<T, VEC> &r, float (&x)[VEC]) {
  if constexpr (T == ANC_BF16) {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {
      x[2 * i] = __uint_as_float(r.q[i] << 16);
      x[2 * i + 1] = __uint_as_float(r.q[i] & 0xFFFF0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = r.q[i];
      if constexpr (VEC == 8) x[4 + i] = r.r[i];
    }
  }
}
template <int T, int VEC> __device__ __forceinline__ Raw<T, VEC> narrow(const float (&x)[VEC]) {
  Raw<T, VEC> r;
  if constexpr (T == ANC_BF16) {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) r.q[i] = bf16_pair(x[2 * i], x[2 * i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      r.q[i] = x[i];
      if constexpr (VEC == 8) r.r[i] = x[4 + i];
    }
  }
  return r;
}

// i / d for i < 2^31 as one multiplication (64-bit division by a value that is not known to the compiler is some hundred instructions):
// m = ceil(2^(31 + s) / d) for the smallest s with 2^s >= d. From d >= 2^(s - 1) + 1 and d < 2^31 follows m < 2^32: 2^(31 + s) / d is at most
// 2^32 - 2^32 / (2^(s - 1) + 1), 2^32 - 3 or less. And m d - 2^(31 + s) < d <= 2^s, so m i / 2^(31 + s) exceeds i / d by less than 1 / d.
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

// ---- host side
constexpr int64_t kMostPieces = (1ll << 31) - 1;     // of one launch (FastDiv)
// Bytes up to which rows go through the caches; through them and past them, us, bf16 rows of 1024 values. A lookup and a copy of it afterwards: 32
// MiB 20.3 and 22.9, 48 30.3 and 32.4, 64 47.7 and 42.2, 128 115 and 96. A gradient after the copy that made its dy: 32 MiB 28.9 both, 64 57 and 47, 128
// 128 and 124. combine_grad by itself is faster past them from 16 MiB on (9.9 and 9.4; 64 MiB 35 and 28), together with the experts' gradient that
// reads its dys from 256 MiB on (335 and 333; 16 MiB 36.3 and 36.9, 64 93.0 and 94.6, 128 173 and 176): the line is between the two.
constexpr int64_t kCached = 64ll << 20;
inline int64_t elem_size(int type) { return type == ANC_F32 ? 4 : 2; }
inline bool type_ok(int type) { return type == ANC_F32 || type == ANC_BF16; }
inline int64_t pieces_of(int64_t H, int64_t vec) { return (H + vec - 1) / vec; }
template <int V> struct Int { static constexpr int value = V; };
template <typename F> inline void with_type(int type, F &&f) {
  if (type == ANC_F32) f(Int<ANC_F32>{}); else f(Int<ANC_BF16>{});
}
template <typename F> inline void with_flag(bool b, F &&f) {
  if (b) f(Int<1>{}); else f(Int<0>{});
}

}  // namespace anc_rows
