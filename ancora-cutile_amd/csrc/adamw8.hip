// AdamW with the moments in 8 bits: per 64 consecutive elements (a row of the tensor's (numel/64, 64) view) m is E4M3 codes and
// v E5M2 codes, each with one E8M0 byte (value = code * 2^(byte - 127)). One sweep over HBM: the moments are widened to fp32, take the
// step of adamw.hip operation by operation, and go back as codes of the new block's scale.
//
// byte = (biased fp32 exponent of the block's largest magnitude) - 7 for m, - 14 for v (at least 1), so that the largest lands in
// [128, 256) of E4M3's 448, in [2^14, 2^15) of E5M2's 57344. v takes the wider range because the update divides by its root: 2^30 and more between
// a block's largest v and its least code is 2^15 between gradients, and a v that is not zero never becomes zero.
//
// Both are stored by stochastic rounding, the code's lower neighbour plus one where the dropped bits and 16 bits of a hash
// of (row, column, seed) carry (v_cvt_sr_fp8_f32 / v_cvt_sr_bf8_f32 with the 16 bits in the upper half of their operand): rounded to nearest, a
// moment that moves by a thousandth a step would stay where it is for ever, since a code's step is an eighth (m) or a quarter (v); this
// way its expectation is the exact moment's. For v that ends at the least code, 2^-31 to 2^-30 of the block's largest: one whose gradients have ended
// stays there while the block's largest does. It also takes a dither of each step's own: a launch whose seed does not move with the steps
// counted on the device is not captured into a graph (300 replays with one dither leave v at 0.12 of what it should be on average, m at 0.72).
// Single elements stray: random gradients of one size, 400 steps: v 23 % rms off the one of 32 bits at beta2 0.95, 29 % at 0.999, m 9 %, the
// update 15 to 18 %.
//
// Bound: 16 1/16 bytes per element (bf16 gradients; read g 2, m 1, v 1, p32 4, write m 1, v 1, p32 4, p16 2, scales) against the 28 of 32-bit
// moments, so little that the arithmetic counts as much: the first form took 173 instructions per element and 179 us for 51.5 M elements (4.6
// TB/s), its three divisions, root and the bookkeeping of codes most of them.
#include "adamw_elem.h"

namespace {

constexpr int kThreads = 256, kVec = 4, kSlabs = 4;
constexpr int kSlab = kThreads * kVec, kBlockElems = kSlab * kSlabs;      // as adamw.hip: anc_adamw_num_blocks
constexpr uint32_t kStateSeed = 0x3C6EF372u;                              // apart from the weights' dither
constexpr uint32_t kInf = 0x7F800000u;
constexpr int64_t kFewBlocks = 2048;                                     // see k_adamw8_multi

__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return a > b ? a : b; }
// The largest of 16 neighbouring lanes, in all of them: rotations within a row of the data-parallel moves.
__device__ __forceinline__ uint32_t max_of_16(uint32_t x) {
#define ANC_ROT(n) x = larger(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x120 + n, 0xF, 0xF, true));
  ANC_ROT(8) ANC_ROT(4) ANC_ROT(2) ANC_ROT(1)
#undef ANC_ROT
  return x;
}
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax, uint32_t top) {
  const uint32_t e = amax >> 23;
  return e > top ? e - top : 1u;
}
// a / b for a b that many elements share, y = 1 / b rounded to nearest: two corrections make the quotient the correctly rounded one (Markstein's
// theorem: the first leaves it within a unit, the remainder of the second is exact), 6 instructions instead of 11. For 0 < |a| < 2^-100 remainders
// leave the range of fp32: those take the plain division (`step_of_four`). Beyond the largest fp32 the last instruction makes infinity of it.
__device__ __forceinline__ float shared_div(float a, float b, float y) {
  float q = a * y;
  q = __builtin_fmaf(__builtin_fmaf(-b, q, a), y, q);
  q = __builtin_fmaf(__builtin_fmaf(-b, q, a), y, q);
  return __builtin_amdgcn_div_fixupf(q, b, a);                            // (infinities, NaN, zeros)
}
// adamw_elem of adamw_elem.h for a lane's four elements, with the bias corrections' reciprocals at hand. (Looking at the moments' least, 51.5 M
// elements, in turn on one card: 146.9 us without, 147.9 with; plain divisions in a branch with all that follows them 148.6.)
template <int FORM>
__device__ __forceinline__ void step_of_four(const anc_f32x4 &g, float (&m)[4], float (&v)[4], float (&p)[4], const anc_adamw_hyper_t &h, float y1, float y2,
                                             float wd, float clip) {
  if constexpr (FORM == ANC_ADAMW_FORM_DIV) {
    float least = __uint_as_float(kInf);                                  // of the magnitudes
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float gs = g[k] * clip;
      m[k] = h.beta1 * m[k] + h.omb1 * gs;
      v[k] = h.beta2 * v[k] + (h.omb2 * gs) * gs;
      least = __builtin_fminf(__builtin_fminf(__builtin_fabsf(m[k]), v[k]), least);
    }
    float mh[4], vh[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      mh[k] = shared_div(m[k], h.bc1, y1);
      vh[k] = shared_div(v[k], h.bc2, y2);
    }
    if (__builtin_expect(least < 0x1p-100f, 0)) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {                                       // (zeros' quotients are right)
        if (m[k] != 0.0f && __builtin_fabsf(m[k]) < 0x1p-100f) mh[k] = m[k] / h.bc1;
        if (v[k] != 0.0f && v[k] < 0x1p-100f) vh[k] = v[k] / h.bc2;
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) p[k] = p[k] - h.lr * (mh[k] / (sqrtf(vh[k]) + h.eps) + wd * p[k]);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) adamw_elem<FORM>(g[k], m[k], v[k], p[k], h, wd, clip);
  }
}

// The hash of anc_sr_hash from its key.
__device__ __forceinline__ uint32_t mixed(uint32_t key) {
  uint32_t h = key * 0x9E3779B1u;
  h ^= h >> 16;
  h *= 0x85EBCA6Bu;
  return h ^ (h >> 13);
}

template <int SLABS> struct Loaded {
  anc_f32x4 g[SLABS], p[SLABS];
  uint32_t m[SLABS], v[SLABS], ms[SLABS], vs[SLABS];
};

// 1024 elements at e (this lane's four of them), loaded in slab j.
template <int FORM, int SR, int SLABS>
__device__ __forceinline__ void adamw8_slab(const anc_adamw8_desc_t &t, const Loaded<SLABS> &in, int j, int64_t e, const anc_adamw_hyper_t &h, float y1,
                                            float y2, float clip, uint32_t seed) {
  const float sm = __uint_as_float(in.ms[j] << 23), sv = __uint_as_float(in.vs[j] << 23);
  const auto ma = __builtin_amdgcn_cvt_pk_f32_fp8((int)in.m[j], false), mb = __builtin_amdgcn_cvt_pk_f32_fp8((int)in.m[j], true);
  const auto va = __builtin_amdgcn_cvt_pk_f32_bf8((int)in.v[j], false), vb = __builtin_amdgcn_cvt_pk_f32_bf8((int)in.v[j], true);
  float mm[4] = {ma[0] * sm, ma[1] * sm, mb[0] * sm, mb[1] * sm};
  float vv[4] = {va[0] * sv, va[1] * sv, vb[0] * sv, vb[1] * sv};
  float pp[4] = {in.p[j].x, in.p[j].y, in.p[j].z, in.p[j].w};
  step_of_four<FORM>(in.g[j], mm, vv, pp, h, y1, y2, t.wd, clip);
  uint32_t am = 0u, av = 0u, ap = 0u;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    am = larger(am, __float_as_uint(mm[k]) & 0x7FFFFFFFu);
    av = larger(av, __float_as_uint(vv[k]));                              // (never negative; a NaN is larger than infinity either way)
    ap = larger(ap, __float_as_uint(pp[k]) & 0x7FFFFFFFu);
  }
  am = max_of_16(am);
  av = max_of_16(av);
  const bool odd = am >= kInf || av >= kInf;                              // something in the block is not finite: it does not count
  if (odd) {
    am = av = 0u;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t a = __float_as_uint(mm[k]) & 0x7FFFFFFFu, b = __float_as_uint(vv[k]);
      am = larger(am, a < kInf ? a : 0u);
      av = larger(av, b < kInf ? b : 0u);
    }
    am = max_of_16(am);
    av = max_of_16(av);
  }
  const uint32_t bm = scale_byte(am, 7u), bv = scale_byte(av, 14u);
  const float um = __uint_as_float((254u - bm) << 23), uv = __uint_as_float((254u - bv) << 23);
  // keys of the hashes: (row * c1) ^ (column * c2) ^ seed, the column's part the same in every slab
  const uint32_t row = (uint32_t)(e >> 6) * 73856093u, col = ((uint32_t)threadIdx.x & 15u) * (4u * 19349663u);
  uint32_t mo = 0u, vo = 0u;
#define ANC_CODE(k)                                                                                        \
  {                                                                                                        \
    const uint32_t d = mixed(row ^ (col + k * 19349663u) ^ (seed ^ kStateSeed));                           \
    mo = (uint32_t)__builtin_amdgcn_cvt_sr_fp8_f32(mm[k] * um, (int)(d << 16), (int)mo, k);                \
    vo = (uint32_t)__builtin_amdgcn_cvt_sr_bf8_f32(vv[k] * uv, (int)(d & 0xFFFF0000u), (int)vo, k);        \
  }
  ANC_CODE(0) ANC_CODE(1) ANC_CODE(2) ANC_CODE(3)
#undef ANC_CODE
  const uint32_t none = ~((vo & 0x7F7F7F7Fu) + 0x7F7F7F7Fu) & 0x80808080u;     // bytes of v that became zero
  if (odd || none != 0u) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (vv[k] > 0.0f && (vo >> (8 * k) & 0xFFu) == 0u) vo |= 1u << (8 * k);
      if (!(__builtin_fabsf(mm[k]) < __uint_as_float(kInf)))
        mo = (mo & ~(0xFFu << (8 * k))) | ((0x7Fu | (__float_as_uint(mm[k]) >> 24 & 0x80u)) << (8 * k));
      if (!(vv[k] < __uint_as_float(kInf))) vo = (vo & ~(0xFFu << (8 * k))) | (0x7Fu << (8 * k));
    }
  }
  uint32_t h2[2];
  if constexpr (SR) {
    uint32_t b[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) b[k] = __float_as_uint(pp[k]) + (mixed(row ^ (col + k * 19349663u) ^ seed) & 0xFFFFu);
    if (ap >= kInf) {
#pragma unroll
      for (int k = 0; k < 4; ++k) b[k] = anc_bf16_sr_bits(pp[k], (uint32_t)(e >> 6), ((uint32_t)e & 63u) + k, seed) << 16;
    }
    h2[0] = __builtin_amdgcn_perm(b[1], b[0], 0x07060302u);
    h2[1] = __builtin_amdgcn_perm(b[3], b[2], 0x07060302u);
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) h2[i] = anc_bf16_rne_bits(pp[2 * i]) | (anc_bf16_rne_bits(pp[2 * i + 1]) << 16);
  }
  anc_st_stream((uint32_t *)((uint8_t *)t.m + e), mo);
  anc_st_stream((uint32_t *)((uint8_t *)t.v + e), vo);
  anc_st_stream((anc_f32x4 *)((float *)t.p32 + e), anc_f32x4{pp[0], pp[1], pp[2], pp[3]});
  anc_st_stream((anc_u32x2 *)((uint16_t *)t.p16 + e), anc_u32x2{h2[0], h2[1]});
  if ((threadIdx.x & 15) == 0) {
    ((uint8_t *)t.ms)[e >> 6] = (uint8_t)bm;
    ((uint8_t *)t.vs)[e >> 6] = (uint8_t)bv;
  }
}

template <int GD, int FORM, int SR, int SLABS>
__device__ __forceinline__ void adamw8_slabs(const anc_adamw8_desc_t &t, int64_t first, const anc_adamw_hyper_t &h, float clip, uint32_t seed) {
  const int64_t base = first + (int64_t)threadIdx.x * kVec;
  Loaded<SLABS> in;
#pragma unroll
  for (int j = 0; j < SLABS; ++j) {
    const int64_t e = base + (int64_t)j * kSlab;
    if (e >= t.n) continue;                                // (n % 64 == 0: 16 lanes live or die together)
    if (GD == ANC_BF16) {
      const anc_u32x2 gb = anc_ld_stream((const anc_u32x2 *)((const uint16_t *)t.g + e));
      in.g[j] = anc_f32x4{__uint_as_float(gb.x << 16), __uint_as_float(gb.x & 0xFFFF0000u), __uint_as_float(gb.y << 16),
                          __uint_as_float(gb.y & 0xFFFF0000u)};
    } else {
      in.g[j] = anc_ld_stream((const anc_f32x4 *)((const float *)t.g + e));
    }
    in.m[j] = anc_ld_stream((const uint32_t *)((const uint8_t *)t.m + e));
    in.v[j] = anc_ld_stream((const uint32_t *)((const uint8_t *)t.v + e));
    in.p[j] = anc_ld_stream((const anc_f32x4 *)((const float *)t.p32 + e));
    in.ms[j] = ((const uint8_t *)t.ms)[e >> 6];
    in.vs[j] = ((const uint8_t *)t.vs)[e >> 6];
  }
  const float y1 = FORM == ANC_ADAMW_FORM_DIV ? 1.0f / h.bc1 : 0.0f, y2 = FORM == ANC_ADAMW_FORM_DIV ? 1.0f / h.bc2 : 0.0f;
#pragma unroll
  for (int j = 0; j < SLABS; ++j) {
    const int64_t e = base + (int64_t)j * kSlab;
    if (e < t.n) adamw8_slab<FORM, SR, SLABS>(t, in, j, e, h, y1, y2, clip, seed);
  }
}

// SLABS = 4: a workgroup takes a whole block of 4096 elements, all of a lane's loads before its arithmetic; 1: a quarter of one, for launches of fewer
// than kFewBlocks blocks, whose last round leaves fewer CUs idle that way. One card, whole blocks and quarters, us: 64 blocks 7.0 and 5.7, 300 10.3 and 7.0,
// 600 13.5 and 10.3 (3.8 TB/s), 1200 21.3 and 17.0, 1600 27.6 and 22.7, 2500 40.5 and 40.0, 5000 73.2 and 74.2, 12576 167 and 166.
template <int FORM, int SR, int SLABS>
__global__ void __launch_bounds__(kThreads)
k_adamw8_multi(const anc_adamw8_desc_t *__restrict__ table, int n_tensors, anc_adamw_hyper_t h, const anc_step_ctl_t *__restrict__ ctl) {
  float clip;
  if (!load_ctl(ctl, clip)) return;
  step_scalars(h, ctl);
  const int64_t blk = (int64_t)(blockIdx.x / (kSlabs / SLABS));
  int lo = 0, hi = n_tensors - 1;                          // last tensor whose first block is <= blk
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (table[mid].blk0 <= blk) lo = mid; else hi = mid - 1;
  }
  const anc_adamw8_desc_t d = table[lo];
  const int64_t first = (blk - d.blk0) * kBlockElems + (int64_t)(blockIdx.x % (kSlabs / SLABS)) * (SLABS * kSlab);
  if (d.g_dtype == ANC_BF16) adamw8_slabs<ANC_BF16, FORM, SR, SLABS>(d, first, h, clip, h.seed_base + d.seed);
  else                       adamw8_slabs<ANC_F32, FORM, SR, SLABS>(d, first, h, clip, h.seed_base + d.seed);
}

}  // namespace

extern "C" int anc_adamw8_multi(uint64_t desc_table, int32_t n_tensors, int64_t total_blocks, const anc_adamw_hyper_t *h, uint64_t ctl,
                                uint64_t stream) {
  ANC_REQUIRE(h != nullptr, "anc_adamw8_multi: null hyper-parameter block");
  ANC_REQUIRE(h->form == ANC_ADAMW_FORM_DIV || h->form == ANC_ADAMW_FORM_IBC, "anc_adamw8_multi: unknown form %d", h->form);
  ANC_REQUIRE((h->sr & ~(ANC_SR_ON | ANC_SR_STEP_SEED)) == 0, "anc_adamw8_multi: sr is a sum of ANC_SR_ON and ANC_SR_STEP_SEED");
  ANC_REQUIRE(h->step_table == 0 || ((h->step_table & 15) == 0 && h->step_cap >= 1),
              "anc_adamw8_multi: step_table must be 16-byte aligned with step_cap >= 1");
  ANC_REQUIRE(ctl != 0 || (h->step_table == 0 && !(h->sr & ANC_SR_STEP_SEED)),
              "anc_adamw8_multi: steps counted on the device need the control block");
  ANC_REQUIRE(desc_table != 0 && (desc_table & 7) == 0 && n_tensors > 0, "anc_adamw8_multi: empty descriptor table");
  ANC_REQUIRE(total_blocks > 0 && total_blocks < (1ll << 31), "anc_adamw8_multi: total_blocks=%lld out of range", (long long)total_blocks);
  if (!(h->sr & ANC_SR_STEP_SEED)) {       // replays would round every moment by one and the same dither, which stops them where they are
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    ANC_HIP(hipStreamIsCapturing(anc_stream(stream), &st));
    ANC_REQUIRE(st == hipStreamCaptureStatusNone, "anc_adamw8_multi: a launch that carries its step's seed cannot be captured into a graph (ANC_SR_STEP_SEED can)");
  }
  const anc_adamw_hyper_t hh = *h;
  AncProfScope prof(ANC_PROF_ADAMW, anc_stream(stream));
  dispatch_form_sr(hh.form, hh.sr & ANC_SR_ON, [&](auto F, auto S) {
    constexpr int f = decltype(F)::value, s = decltype(S)::value;
    const auto *tab = (const anc_adamw8_desc_t *)desc_table;
    const auto *c = (const anc_step_ctl_t *)ctl;
    if (total_blocks < kFewBlocks)
      hipLaunchKernelGGL((k_adamw8_multi<f, s, 1>), dim3((unsigned)(total_blocks * kSlabs)), dim3(kThreads), 0, anc_stream(stream), tab, (int)n_tensors, hh, c);
    else
      hipLaunchKernelGGL((k_adamw8_multi<f, s, kSlabs>), dim3((unsigned)total_blocks), dim3(kThreads), 0, anc_stream(stream), tab, (int)n_tensors, hh, c);
  });
  ANC_LAUNCH_CHECK();
  return ANC_OK;
}
