// AdamW with the moments in 8 bits: per 64 consecutive elements (a row of the tensor's (numel/64, 64) view) m is E4M3 codes and
// v E5M2 codes, each with one E8M0 byte (value = code * 2^(byte - 127)). One sweep over HBM: the moments are widened to fp32, take the
// step of adamw.hip operation by operation, and go back as codes of the new block's scale.
//
// byte = (biased fp32 exponent of the block's largest magnitude) - 7 for m, - 14 for v (at least 1), so that the largest lands in
// [128, 256) of E4M3's 448, in [2^14, 2^15) of E5M2's 57344. v takes the wider range because the update divides by its root: 2^31 between
// a block's largest v and its least normal one is 2^15 between gradients, and a v that is not zero never becomes zero.
//
// Both are stored by stochastic rounding, the code's lower neighbour plus one where the dropped bits and 16 bits of a hash
// of (row, column, seed) carry: rounded to nearest, a moment that moves by a thousandth a step would stay where it is for ever, since a code's
// step is an eighth (m) or a quarter (v); this way its expectation is the exact moment's.
//
// HBM-bound: 16 1/16 bytes per element (bf16 gradients; read g 2, m 1, v 1, p32 4, write m 1, v 1, p32 4, p16 2, scales) against the
// 28 of 32-bit moments.
#include "adamw_elem.h"

namespace {

constexpr int kThreads = 256, kVec = 4, kUnroll = 4;
constexpr int kSlab = kThreads * kVec, kBlockElems = kSlab * kUnroll;    // as adamw.hip: anc_adamw_num_blocks
constexpr uint32_t kStateSeed = 0x3C6EF372u;                              // apart from the weights' dither

// The largest of 16 neighbouring lanes, in all of them: rotations within a row of the data-parallel moves.
__device__ __forceinline__ uint32_t max_of_16(uint32_t x) {
#define ANC_ROT(n) { const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x120 + n, 0xF, 0xF, true); x = x > o ? x : o; }
  ANC_ROT(8) ANC_ROT(4) ANC_ROT(2) ANC_ROT(1)
#undef ANC_ROT
  return x;
}
// Magnitude bits of a finite number, 0 of any other: a NaN does not decide its block's scale.
__device__ __forceinline__ uint32_t finite_bits(float x) {
  const uint32_t b = __float_as_uint(x) & 0x7FFFFFFFu;
  return b < 0x7F800000u ? b : 0u;
}
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax, uint32_t top) {
  const uint32_t e = amax >> 23;
  return e > top ? e - top : 1u;
}
// Code (without sign) of x >= 0 times the power of two `up`; MANT mantissa bits, exponent field 1 stands for 2^(1 + BASE - 127), dither
// of 16 bits. A subnormal code's steps are those of the least normal binade, into which the sum moves it. NaN and infinity: 0x7F.
template <int MANT, int BASE>
__device__ __forceinline__ uint32_t code_of(float x, float up, uint32_t dither) {
  constexpr int kDrop = 23 - MANT;
  const float low = __uint_as_float((uint32_t)(BASE + 1) << 23);
  const float y = x * up;
  const bool small = y < low;
  const uint32_t b = __float_as_uint(small ? y + low : y) + (dither << (kDrop - 16));
  const uint32_t c = (b >> kDrop) - ((uint32_t)(small ? BASE + 1 : BASE) << MANT);
  return x < __uint_as_float(0x7F800000u) ? c : 0x7Fu;
}

template <int GD, int FORM, int SR>
__device__ __forceinline__ void adamw8_block(const anc_adamw8_desc_t &t, int64_t blk, const anc_adamw_hyper_t &h, float clip, uint32_t seed) {
  const int64_t base = blk * kBlockElems + (int64_t)threadIdx.x * kVec;
  const uint8_t *tm = (const uint8_t *)t.m, *tv = (const uint8_t *)t.v, *tms = (const uint8_t *)t.ms, *tvs = (const uint8_t *)t.vs;
  anc_f32x4 g4[kUnroll], p4[kUnroll];
  uint32_t m4[kUnroll], v4[kUnroll], ms[kUnroll], vs[kUnroll];
  bool live[kUnroll];
#pragma unroll
  for (int j = 0; j < kUnroll; ++j) {
    const int64_t e = base + (int64_t)j * kSlab;
    live[j] = e < t.n;                                     // (n % 64 == 0: 16 lanes live or die together)
    if (live[j]) {
      if (GD == ANC_BF16) {
        const anc_u32x2 gb = anc_ld_stream((const anc_u32x2 *)((const uint16_t *)t.g + e));
        g4[j] = anc_f32x4{__uint_as_float(gb.x << 16), __uint_as_float(gb.x & 0xFFFF0000u), __uint_as_float(gb.y << 16),
                          __uint_as_float(gb.y & 0xFFFF0000u)};
      } else {
        g4[j] = anc_ld_stream((const anc_f32x4 *)((const float *)t.g + e));
      }
      m4[j] = anc_ld_stream((const uint32_t *)(tm + e));
      v4[j] = anc_ld_stream((const uint32_t *)(tv + e));
      p4[j] = anc_ld_stream((const anc_f32x4 *)((const float *)t.p32 + e));
      ms[j] = tms[e >> 6];
      vs[j] = tvs[e >> 6];
    }
  }
#pragma unroll
  for (int j = 0; j < kUnroll; ++j) {
    if (!live[j]) continue;
    const int64_t e = base + (int64_t)j * kSlab;
    const float gg[4] = {g4[j].x, g4[j].y, g4[j].z, g4[j].w};
    float pp[4] = {p4[j].x, p4[j].y, p4[j].z, p4[j].w};
    const float sm = __uint_as_float(ms[j] << 23), sv = __uint_as_float(vs[j] << 23);
    const auto ma = __builtin_amdgcn_cvt_pk_f32_fp8((int)m4[j], false), mb = __builtin_amdgcn_cvt_pk_f32_fp8((int)m4[j], true);
    const auto va = __builtin_amdgcn_cvt_pk_f32_bf8((int)v4[j], false), vb = __builtin_amdgcn_cvt_pk_f32_bf8((int)v4[j], true);
    float mm[4] = {ma[0] * sm, ma[1] * sm, mb[0] * sm, mb[1] * sm};
    float vv[4] = {va[0] * sv, va[1] * sv, vb[0] * sv, vb[1] * sv};
    uint32_t hb[4], am = 0u, av = 0u;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      adamw_elem<FORM>(gg[k], mm[k], vv[k], pp[k], h, t.wd, clip);
      const uint64_t i = (uint64_t)(e + k);
      hb[k] = SR ? anc_bf16_sr_bits(pp[k], (uint32_t)(i >> 6), (uint32_t)(i & 63u), seed) : anc_bf16_rne_bits(pp[k]);
      const uint32_t a = finite_bits(mm[k]), b = finite_bits(vv[k]);
      am = am > a ? am : a;
      av = av > b ? av : b;
    }
    const uint32_t bm = scale_byte(max_of_16(am), 7u), bv = scale_byte(max_of_16(av), 14u);
    const float um = __uint_as_float((254u - bm) << 23), uv = __uint_as_float((254u - bv) << 23);
    uint32_t mo = 0u, vo = 0u;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint64_t i = (uint64_t)(e + k);
      const uint32_t d = anc_sr_hash((uint32_t)(i >> 6), (uint32_t)(i & 63u), seed ^ kStateSeed);
      const uint32_t cm = code_of<3, 120>(__builtin_fabsf(mm[k]), um, d & 0xFFFFu) | ((__float_as_uint(mm[k]) >> 24) & 0x80u);
      const uint32_t cv = code_of<2, 112>(vv[k], uv, d >> 16);
      mo |= cm << (8 * k);
      vo |= (vv[k] > 0.0f && cv == 0u ? 1u : cv) << (8 * k);
    }
    anc_st_stream((uint32_t *)((uint8_t *)t.m + e), mo);
    anc_st_stream((uint32_t *)((uint8_t *)t.v + e), vo);
    anc_st_stream((anc_f32x4 *)((float *)t.p32 + e), anc_f32x4{pp[0], pp[1], pp[2], pp[3]});
    anc_st_stream((anc_u32x2 *)((uint16_t *)t.p16 + e), anc_u32x2{(hb[0] & 0xFFFFu) | (hb[1] << 16), (hb[2] & 0xFFFFu) | (hb[3] << 16)});
    if ((threadIdx.x & 15) == 0) {
      ((uint8_t *)t.ms)[e >> 6] = (uint8_t)bm;
      ((uint8_t *)t.vs)[e >> 6] = (uint8_t)bv;
    }
  }
}

template <int FORM, int SR>
__global__ void __launch_bounds__(kThreads)
k_adamw8_multi(const anc_adamw8_desc_t *__restrict__ table, int n_tensors, anc_adamw_hyper_t h, const anc_step_ctl_t *__restrict__ ctl) {
  float clip;
  if (!load_ctl(ctl, clip)) return;
  step_scalars(h, ctl);
  const int64_t blk = (int64_t)blockIdx.x;
  int lo = 0, hi = n_tensors - 1;                          // last tensor whose first block is <= blk
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (table[mid].blk0 <= blk) lo = mid; else hi = mid - 1;
  }
  const anc_adamw8_desc_t d = table[lo];
  if (d.g_dtype == ANC_BF16) adamw8_block<ANC_BF16, FORM, SR>(d, blk - d.blk0, h, clip, h.seed_base + d.seed);
  else                       adamw8_block<ANC_F32, FORM, SR>(d, blk - d.blk0, h, clip, h.seed_base + d.seed);
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
  const anc_adamw_hyper_t hh = *h;
  AncProfScope prof(ANC_PROF_ADAMW, anc_stream(stream));
  dispatch_form_sr(hh.form, hh.sr & ANC_SR_ON, [&](auto F, auto S) {
    constexpr int f = decltype(F)::value, s = decltype(S)::value;
    hipLaunchKernelGGL((k_adamw8_multi<f, s>), dim3((unsigned)total_blocks), dim3(kThreads), 0, anc_stream(stream),
                       (const anc_adamw8_desc_t *)desc_table, (int)n_tensors, hh, (const anc_step_ctl_t *)ctl);
  });
  ANC_LAUNCH_CHECK();
  return ANC_OK;
}
