// Root-mean-square norm of rows with the residual's addition in front of it and, for products in 8 bits, MXFP8 rows behind it; and its
// backward pass. The reference's layers run it between the optimizer's weights; its gain is one of AdamW's tensors.
//
//   s = x + residual,  r = 1 / sqrt(mean(s^2) + eps),  y = s r gain                                (all in fp32, one rounding per output)
//   MXFP8: per 32 elements of a row byte = (biased exponent of the largest |y|) - 7 (0 below 7), element = E4M3(y 2^(127 - byte)): the
//   format of quant.hip with the blocks along the row, which is the axis that a product with the weights runs over
//   a = dy gain,  dx = r (a - s r^2 mean(a s)) + carry,  dgain = sum over rows of dy s r
//
// HBM-bound. A row is held in registers by 16, 64 or 256 lanes (backwards up to 512), 8 elements (16 bytes of bf16) to a piece, so that it is read once.
// The gain's gradient: workgroups add up their rows in registers, then their groups of lanes through LDS, and leave one fp32 row each; a
// second launch adds those in a fixed order. The bits are a function of the inputs and the shape.
#include "rows.h"

namespace {

using anc_rows::bf16_pair;
constexpr int kThreads = 256;
constexpr int kGradThreads = 512;       // of the backward pass: twice the wavefronts to a partial row of dgain
constexpr int kMostRows = 512;          // partial rows of dgain

template <int T> struct Eight;
template <> struct Eight<ANC_BF16> { anc_u32x4 q; };
template <> struct Eight<ANC_F32> { anc_f32x4 q, r; };
template <int T> __device__ __forceinline__ Eight<T> load8(uint64_t p, int64_t e) {
  if constexpr (T == ANC_BF16) return {*(const anc_u32x4 *)((const uint16_t *)p + e)};
  else return {*(const anc_f32x4 *)((const float *)p + e), *(const anc_f32x4 *)((const float *)p + e + 4)};
}
template <int T> __device__ __forceinline__ void widen(const Eight<T> &v, float (&f)[8]) {
  if constexpr (T == ANC_BF16) {
    const uint32_t w[4] = {v.q.x, v.q.y, v.q.z, v.q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[i] = v.q[i];
      f[4 + i] = v.r[i];
    }
  }
}
template <int T> __device__ __forceinline__ void store8(uint64_t p, int64_t e, const float (&f)[8]) {
  if constexpr (T == ANC_BF16) {
    *(anc_u32x4 *)((uint16_t *)p + e) = anc_u32x4{bf16_pair(f[0], f[1]), bf16_pair(f[2], f[3]), bf16_pair(f[4], f[5]), bf16_pair(f[6], f[7])};
  } else {
    *(anc_f32x4 *)((float *)p + e) = anc_f32x4{f[0], f[1], f[2], f[3]};
    *(anc_f32x4 *)((float *)p + e + 4) = anc_f32x4{f[4], f[5], f[6], f[7]};
  }
}

// Sum over the LPR lanes of a row, in all of them, in a fixed order. LPR > 64: every lane of the workgroup calls it; lds: a float per wavefront, two
// sets in turn (`odd`), so that one barrier parts a call from the one before it.
template <int LPR> __device__ __forceinline__ float row_sum(float v, float *lds, int odd = 0) {
#pragma unroll
  for (int off = LPR == 16 ? 8 : 32; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
  if constexpr (LPR > 64) {
    lds += odd * (kGradThreads / 64);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    const float *w = lds + threadIdx.x / LPR * (LPR / 64);
    if constexpr (LPR == 128) v = w[0] + w[1];
    else if constexpr (LPR == 256) v = (w[0] + w[1]) + (w[2] + w[3]);
    else v = ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
  }
  return v;
}

struct NormArgs {
  uint64_t x, residual, gain, y, scale, total, rstd;
  int64_t T;
  int H;
  float eps;
};
constexpr int kMx8 = 2;                 // beside ANC_F32 and ANC_BF16

template <int XT, int ST, int GT, int OT, bool RES, int LPR, int CH>
__global__ void __launch_bounds__(kThreads) k_rms_norm(NormArgs a) {
  __shared__ float lds[4];
  const int sub = (int)threadIdx.x % LPR;
  const int64_t row = (int64_t)blockIdx.x * (kThreads / LPR) + (int)threadIdx.x / LPR;
  const bool live = row < a.T;                        // (a wavefront's other rows still take part in its shuffles)
  const int64_t base = (live ? row : 0) * a.H;
  Eight<XT> x8[CH];
  Eight<ST> r8[CH];
  Eight<GT> g8[CH];
  bool on[CH];
#pragma unroll
  for (int j = 0; j < CH; ++j) {
    const int col = (sub + j * LPR) * 8;
    on[j] = live && col < a.H;
    if (on[j]) {
      x8[j] = load8<XT>(a.x, base + col);
      if constexpr (RES) r8[j] = load8<ST>(a.residual, base + col);
      g8[j] = load8<GT>(a.gain, col);
    }
  }
  float s[CH][8], sum = 0.0f;
#pragma unroll
  for (int j = 0; j < CH; ++j) {
    if (!on[j]) continue;
    widen<XT>(x8[j], s[j]);
    if constexpr (RES) {
      float r[8];
      widen<ST>(r8[j], r);
#pragma unroll
      for (int k = 0; k < 8; ++k) s[j][k] += r[k];
      store8<ST>(a.total, base + (sub + j * LPR) * 8, s[j]);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) sum = __builtin_fmaf(s[j][k], s[j][k], sum);
  }
  sum = row_sum<LPR>(sum, lds);
  const float r = 1.0f / sqrtf(sum / (float)a.H + a.eps);
  if (a.rstd != 0 && live && sub == 0) ((float *)a.rstd)[row] = r;
#pragma unroll
  for (int j = 0; j < CH; ++j) {
    if (!on[j]) continue;
    const int64_t at = base + (sub + j * LPR) * 8;
    float y[8], g[8];
    widen<GT>(g8[j], g);
#pragma unroll
    for (int k = 0; k < 8; ++k) y[k] = s[j][k] * r * g[k];
    if constexpr (OT != kMx8) {
      store8<OT>(a.y, at, y);
    } else {
      uint32_t amax = 0u;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t b = __float_as_uint(y[k]) & 0x7FFFFFFFu;
        amax = amax > b ? amax : b;
      }
      // four neighbouring lanes hold a block (H % 32 == 0: all of them or none)
      uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)amax, 0xB1, 0xF, 0xF, true);      // lane ^ 1
      amax = amax > o ? amax : o;
      o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)amax, 0x4E, 0xF, 0xF, true);                // lane ^ 2
      amax = amax > o ? amax : o;
      const uint32_t ea = amax >> 23, byte = ea >= 7u ? ea - 7u : 0u;
      const float up = __uint_as_float((254u - byte) << 23);
      uint32_t w[2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
        w[h] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[4 * h + 2] * up, y[4 * h + 3] * up,
                                                         __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * h] * up, y[4 * h + 1] * up, 0, false), true);
      if (ea == 255u) {                                // something is not finite: those elements become NaN codes
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if ((__float_as_uint(y[k]) & 0x7F800000u) == 0x7F800000u)
            w[k >> 2] = (w[k >> 2] & ~(0xFFu << (8 * (k & 3)))) | ((0x7Fu | ((__float_as_uint(y[k]) >> 24) & 0x80u)) << (8 * (k & 3)));
      }
      *(anc_u32x2 *)((uint8_t *)a.y + at) = anc_u32x2{w[0], w[1]};
      if ((threadIdx.x & 3) == 0) ((uint8_t *)a.scale)[at >> 5] = (uint8_t)byte;
    }
  }
}

struct GradArgs {
  uint64_t dy, x, gain, rstd, carry, dx, dgain, parts;
  int64_t T;
  int H, rows, accumulate;              // rows of dgain in parts: the grid
};

// One row's pieces in registers, as they lie in memory.
template <int DT, int ST, bool CARRY, int CH> struct GradRow {
  Eight<DT> d[CH];
  Eight<ST> s[CH], c[CARRY ? CH : 1];
  float r;
};

// Group g of workgroup b takes rows b * groups + g, then every rows * groups further. The gain is kept, or read again where four or more
// pieces leave no room for it. (8192 rows of 1024 in bf16 with carry, both launches, 64 lanes to a row: workgroups of 256 lanes 16.2 us, of 512 15.2; 256
// partial rows 16.1; the next row's loads ahead of this row's sums 16.7: the wavefronts that their registers displace were worth more.)
template <int DT, int ST, int WT, bool CARRY, int LPR, int CH>
__global__ void __launch_bounds__(kGradThreads, 1) k_rms_norm_grad(GradArgs a) {
  constexpr int kGroups = kGradThreads / LPR;
  constexpr bool kKeep = CH < 4;
  __shared__ float lds[2 * kGradThreads / 64];
  __shared__ float sums[kGroups > 1 ? kGroups * LPR * CH * 8 : 1];
  const int sub = (int)threadIdx.x % LPR, group = (int)threadIdx.x / LPR;
  Eight<WT> kept[kKeep ? CH : 1];
  float dg[CH][8];
  auto gain = [&](int j) {
    if constexpr (kKeep) return kept[j];
    else return load8<WT>(a.gain, (sub + j * LPR) * 8);
  };
  using Row = GradRow<DT, ST, CARRY, CH>;
  auto fetch = [&](int64_t row, Row &v) {
    if (row >= a.T) return;
    v.r = ((const float *)a.rstd)[row];
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      const int col = (sub + j * LPR) * 8;
      if (col >= a.H) continue;
      v.d[j] = load8<DT>(a.dy, row * a.H + col);
      v.s[j] = load8<ST>(a.x, row * a.H + col);
      if constexpr (CARRY) v.c[j] = load8<ST>(a.carry, row * a.H + col);
    }
  };
  Row now;
  int odd = 0;
#pragma unroll
  for (int j = 0; j < CH; ++j) {
    const int col = (sub + j * LPR) * 8;
    if constexpr (kKeep) {
      if (col < a.H) kept[j] = load8<WT>(a.gain, col);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) dg[j][k] = 0.0f;
  }
  for (int64_t row0 = (int64_t)blockIdx.x * kGroups; row0 < a.T; row0 += (int64_t)a.rows * kGroups) {
    const int64_t row = row0 + group;
    const bool live = row < a.T;                      // (a wavefront's other rows still take part in its shuffles)
    fetch(row, now);
    const float r = now.r;
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      if (!live || (sub + j * LPR) * 8 >= a.H) continue;
      float d[8], s[8], g[8];
      widen<DT>(now.d[j], d);
      widen<ST>(now.s[j], s);
      widen<WT>(gain(j), g);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float xh = s[k] * r;
        dg[j][k] = __builtin_fmaf(d[k], xh, dg[j][k]);
        sum = __builtin_fmaf(d[k] * g[k], xh, sum);
      }
    }
    const float c = row_sum<LPR>(sum, lds, odd) / (float)a.H;
    odd ^= 1;
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      if (!live || (sub + j * LPR) * 8 >= a.H) continue;
      float d[8], s[8], g[8], o[8];
      widen<DT>(now.d[j], d);
      widen<ST>(now.s[j], s);
      widen<WT>(gain(j), g);
#pragma unroll
      for (int k = 0; k < 8; ++k) o[k] = r * (d[k] * g[k] - s[k] * r * c);
      if constexpr (CARRY) {
        float f[8];
        widen<ST>(now.c[j], f);
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] += f[k];
      }
      store8<ST>(a.dx, row * a.H + (sub + j * LPR) * 8, o);
    }
  }
  // the groups' sums in ascending order
  if constexpr (kGroups > 1) {
#pragma unroll
    for (int j = 0; j < CH; ++j)
#pragma unroll
      for (int k = 0; k < 8; ++k) sums[group * LPR * CH * 8 + (sub + j * LPR) * 8 + k] = dg[j][k];
    __syncthreads();
  }
  float *out = a.rows > 1 ? (float *)a.parts + (int64_t)blockIdx.x * a.H : (float *)a.dgain;
  const bool onto = a.rows == 1 && a.accumulate;
  if constexpr (kGroups > 1) {
    for (int col = (int)threadIdx.x; col < a.H; col += kGradThreads) {
      float v = sums[col];
#pragma unroll
      for (int q = 1; q < kGroups; ++q) v += sums[q * LPR * CH * 8 + col];
      out[col] = onto ? out[col] + v : v;
    }
  } else {
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      const int col = (sub + j * LPR) * 8;
      if (col >= a.H) continue;
      if (onto) {
        float f[8];
        widen<ANC_F32>(load8<ANC_F32>((uint64_t)out, col), f);
#pragma unroll
        for (int k = 0; k < 8; ++k) dg[j][k] += f[k];
      }
      store8<ANC_F32>((uint64_t)out, col, dg[j]);
    }
  }
}

// dgain (+)= the sum of `rows` rows: 32 columns, a line, to a workgroup, 64 groups of 8 lanes taking every 64th row, all their loads under way
// at once. (Both launches, us: half lines and loads as they come 15.1 at 3000 x 2048, 18.0 at 500 x 8192; lines 14.5, 17.0; at once 12.7, 16.8; the partial rows
// stored 16 bytes a lane where a row is a workgroup's 12.7, 12.9.)
constexpr int kSumThreads = 512;
__global__ void __launch_bounds__(kSumThreads) k_gain_sum(const float *parts, float *dgain, int rows, int H, int accumulate) {
  __shared__ float sums[64][33];
  const int c8 = (int)threadIdx.x & 7, q = (int)threadIdx.x >> 3, col = (int)blockIdx.x * 32 + c8 * 4;
  anc_f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
  if (col < H) {
    anc_f32x4 p[kMostRows / 64];                      // (all under way at once)
#pragma unroll
    for (int i = 0; i < kMostRows / 64; ++i)
      p[i] = q + 64 * i < rows ? *(const anc_f32x4 *)(parts + (int64_t)(q + 64 * i) * H + col) : anc_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < kMostRows / 64; ++i) v = anc_f32x4{v.x + p[i].x, v.y + p[i].y, v.z + p[i].z, v.w + p[i].w};
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) sums[q][c8 * 4 + k] = v[k];
  __syncthreads();
  // 16 lanes to a column: four rows each, then across the lanes
  const int c = (int)threadIdx.x >> 4, part = (int)threadIdx.x & 15;
  float t = ((sums[part][c] + sums[part + 16][c]) + sums[part + 32][c]) + sums[part + 48][c];
#pragma unroll
  for (int off = 8; off >= 1; off >>= 1) t += __shfl_xor(t, off, 64);
  const int out = (int)blockIdx.x * 32 + c;
  if (part == 0 && out < H) dgain[out] = accumulate ? dgain[out] + t : t;
}

constexpr int kWidest = 16384;
template <int V> struct IC { static constexpr int value = V; };
template <typename F> void with_type(int t, F &&f) {
  if (t == ANC_BF16) f(IC<ANC_BF16>{}); else f(IC<ANC_F32>{});
}
// Lanes per row and pieces per lane.
template <typename F> void with_layout(int H, F &&f) {
  const int pieces = H / 8;
  if (pieces <= 16) f(IC<16>{}, IC<1>{});
  else if (pieces <= 32) f(IC<16>{}, IC<2>{});
  else if (pieces <= 64) f(IC<64>{}, IC<1>{});
  else if (pieces <= 128) f(IC<64>{}, IC<2>{});
  else if (pieces <= 256) f(IC<64>{}, IC<4>{});
  else if (pieces <= 512) f(IC<256>{}, IC<2>{});
  else if (pieces <= 1024) f(IC<256>{}, IC<4>{});
  else f(IC<256>{}, IC<8>{});
}
// The same for the backward pass, whose lanes hold three rows' pieces and dgain's sums: fewer of them to a lane, so that two workgroups or more fit a
// CU. (Both launches, us, half as many lanes or less and these: 8192 x 1024 15.4, 15.1; 3000 x 2048 17.1, 15.1; 8000 x 16384 260, 242; but 4096
// x 4096 with twice these 34.2, 33.2.)
template <typename F> void with_grad_layout(int H, F &&f) {
  const int pieces = H / 8;
  if (pieces <= 16) f(IC<16>{}, IC<1>{});
  else if (pieces <= 32) f(IC<16>{}, IC<2>{});
  else if (pieces <= 64) f(IC<64>{}, IC<1>{});
  else if (pieces <= 128) f(IC<128>{}, IC<1>{});
  else if (pieces <= 256) f(IC<256>{}, IC<1>{});
  else if (pieces <= 512) f(IC<256>{}, IC<2>{});
  else if (pieces <= 1024) f(IC<512>{}, IC<2>{});
  else f(IC<512>{}, IC<4>{});
}
int grad_lanes(int64_t H) { return H <= 256 ? 16 : H <= 512 ? 64 : H <= 1024 ? 128 : H <= 4096 ? 256 : 512; }
int lanes_of(int64_t H) { return H <= 256 ? 16 : H <= 2048 ? 64 : 256; }
bool width_ok(int64_t H) { return H > 0 && H % 8 == 0 && H <= kWidest; }
bool type_ok(int t) { return t == ANC_F32 || t == ANC_BF16; }
int64_t elem(int t) { return t == ANC_BF16 ? 2 : 4; }
// Partial rows of dgain: two rows of the batch per group of lanes at least, as many workgroups as keep the memory busy at most, all with
// as many rows as the fullest.
int64_t parts_of(int64_t T, int64_t H) {
  const int64_t groups = kGradThreads / grad_lanes(H), most = kMostRows * groups;
  const int64_t each = T <= 2 * most ? 2 : (T + most - 1) / most, n = (T + each * groups - 1) / (each * groups);
  return n < 1 ? 1 : n;
}

}  // namespace

extern "C" int anc_rms_norm(uint64_t x, int x_type, uint64_t residual, int stream_type, uint64_t gain, int gain_type, int64_t T, int64_t H,
                            float eps, uint64_t y, int y_type, uint64_t scale, uint64_t total, uint64_t rstd, uint64_t stream) {
  ANC_REQUIRE(type_ok(x_type) && type_ok(stream_type) && type_ok(gain_type) && (type_ok(y_type) || y_type == ANC_MXFP8),
              "anc_rms_norm: bad types (x %d, stream %d, gain %d, y %d)", x_type, stream_type, gain_type, y_type);
  ANC_REQUIRE(width_ok(H), "anc_rms_norm: rows of %lld: a multiple of 8 up to %d", (long long)H, kWidest);
  ANC_REQUIRE(T >= 0 && T < (1ll << 31), "anc_rms_norm: %lld rows", (long long)T);
  ANC_REQUIRE(T * lanes_of(H) <= (1ll << 32) - kThreads, "anc_rms_norm: %lld rows of %lld: too large for one call", (long long)T, (long long)H);
  if (T == 0) return ANC_OK;
  const bool mx8 = y_type == ANC_MXFP8;
  ANC_REQUIRE(x && gain && y && (scale != 0) == mx8 && (residual != 0) == (total != 0),
              "anc_rms_norm: null device pointer (scale goes with 8-bit rows, total with residual)");
  ANC_REQUIRE(!mx8 || H % 32 == 0, "anc_rms_norm: 8-bit rows of %lld: a multiple of 32", (long long)H);
  ANC_REQUIRE(((x | residual | gain | y | total) & 15) == 0 && (rstd & 3) == 0, "anc_rms_norm: misaligned pointers");
  const int64_t n = T * H;
  // (a workgroup reads its rows before it writes them: total may be the residual itself, y or total the x of the same type)
  const AncSpan out[4] = {{y, n * (mx8 ? 1 : elem(y_type))}, {total, total ? n * elem(stream_type) : 0}, {scale, mx8 ? n / 32 : 0}, {rstd, rstd ? 4 * T : 0}};
  const AncSpan in[3] = {{x, n * elem(x_type)}, {residual, residual ? n * elem(stream_type) : 0}, {gain, H * elem(gain_type)}};
  ANC_REQUIRE(anc_outputs_apart({out[0], out[1], out[2], out[3]}, 4), "anc_rms_norm: outputs overlap");
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 3; ++j) {
      const bool same = out[i].at == in[j].at && out[i].bytes == in[j].bytes && i < 2 && j < 2 && !(i == 0 && mx8);
      ANC_REQUIRE(same || anc_apart(out[i].at, out[i].bytes, in[j].at, in[j].bytes), "anc_rms_norm: an output overlaps an input");
    }
  const NormArgs a{x, residual, gain, y, scale, total, rstd, T, (int)H, eps};
  hipStream_t s = anc_stream(stream);
  AncProfScope prof(ANC_PROF_MISC, s);
  with_layout((int)H, [&](auto L, auto C) {
    constexpr int lpr = decltype(L)::value, ch = decltype(C)::value;
    const unsigned grid = (unsigned)((T + kThreads / lpr - 1) / (kThreads / lpr));
    with_type(x_type, [&](auto X) { with_type(stream_type, [&](auto S) { with_type(gain_type, [&](auto G) {
      constexpr int xt = decltype(X)::value, st = decltype(S)::value, gt = decltype(G)::value;
      auto go = [&](auto O) {
        constexpr int ot = decltype(O)::value;
        if (residual) hipLaunchKernelGGL((k_rms_norm<xt, st, gt, ot, true, lpr, ch>), dim3(grid), dim3(kThreads), 0, s, a);
        else hipLaunchKernelGGL((k_rms_norm<xt, ANC_BF16, gt, ot, false, lpr, ch>), dim3(grid), dim3(kThreads), 0, s, a);
      };
      if (mx8) go(IC<kMx8>{});
      else if (y_type == ANC_BF16) go(IC<ANC_BF16>{});
      else go(IC<ANC_F32>{});
    }); }); });
  });
  ANC_LAUNCH_CHECK();
  return ANC_OK;
}

extern "C" int64_t anc_rms_norm_grad_workspace_bytes(int64_t T, int64_t H) {
  if (!width_ok(H) || T < 0 || T >= (1ll << 31)) {
    anc_set_error("anc_rms_norm_grad_workspace_bytes: %lld rows of %lld", (long long)T, (long long)H);
    return -1;
  }
  // (fewer rows than T may want more partial rows than T does, never more than at two rows each)
  const int64_t per = 2 * (kGradThreads / grad_lanes(H)), n = (T + per - 1) / per;
  return (n < 1 ? 1 : n > kMostRows ? kMostRows : n) * H * 4;
}

extern "C" int anc_rms_norm_grad(uint64_t dy, int dy_type, uint64_t x, int stream_type, uint64_t gain, int gain_type, uint64_t rstd,
                                 uint64_t carry, int64_t T, int64_t H, uint64_t dx, uint64_t dgain, int accumulate, uint64_t workspace,
                                 int64_t workspace_bytes, uint64_t stream) {
  ANC_REQUIRE(type_ok(dy_type) && type_ok(stream_type) && type_ok(gain_type), "anc_rms_norm_grad: bad types (dy %d, stream %d, gain %d)",
              dy_type, stream_type, gain_type);
  ANC_REQUIRE(width_ok(H), "anc_rms_norm_grad: rows of %lld: a multiple of 8 up to %d", (long long)H, kWidest);
  ANC_REQUIRE(T >= 0 && T < (1ll << 31), "anc_rms_norm_grad: %lld rows", (long long)T);
  ANC_REQUIRE(gain && dgain && (T == 0 || (dy && x && rstd && dx)), "anc_rms_norm_grad: null device pointer");
  ANC_REQUIRE(((dy | x | gain | carry | dx | dgain | workspace) & 15) == 0 && (rstd & 3) == 0, "anc_rms_norm_grad: misaligned pointers");
  const int64_t need = parts_of(T, H) * H * 4, n = T * H;
  ANC_REQUIRE(workspace != 0 && workspace_bytes >= need, "anc_rms_norm_grad: workspace holds %lld bytes, %lld needed",
              (long long)workspace_bytes, (long long)need);
  const AncSpan out[3] = {{dx, n * elem(stream_type)}, {dgain, 4 * H}, {workspace, need}};
  const AncSpan in[5] = {{dy, n * elem(dy_type)}, {x, n * elem(stream_type)}, {carry, carry ? n * elem(stream_type) : 0}, {gain, H * elem(gain_type)}, {rstd, 4 * T}};
  ANC_REQUIRE(anc_outputs_apart({out[0], out[1], out[2]}, 3), "anc_rms_norm_grad: outputs or workspace overlap");
  for (int i = 0; i < 3; ++i)
    for (int j = 0; j < 5; ++j) {                     // (dx may be dy, x or carry itself)
      const bool same = i == 0 && j < 3 && out[0].at == in[j].at && out[0].bytes == in[j].bytes;
      ANC_REQUIRE(same || anc_apart(out[i].at, out[i].bytes, in[j].at, in[j].bytes), "anc_rms_norm_grad: an output or the workspace overlaps an input");
    }
  GradArgs a{dy, x, gain, rstd, carry, dx, dgain, workspace, T, (int)H, (int)parts_of(T, H), accumulate != 0};
  hipStream_t s = anc_stream(stream);
  AncProfScope prof(ANC_PROF_MISC, s);
  with_grad_layout((int)H, [&](auto L, auto C) {
    constexpr int lpr = decltype(L)::value, ch = decltype(C)::value;
    with_type(dy_type, [&](auto D) { with_type(stream_type, [&](auto S) { with_type(gain_type, [&](auto G) {
      constexpr int dt = decltype(D)::value, st = decltype(S)::value, gt = decltype(G)::value;
      if (carry) hipLaunchKernelGGL((k_rms_norm_grad<dt, st, gt, true, lpr, ch>), dim3((unsigned)a.rows), dim3(kGradThreads), 0, s, a);
      else hipLaunchKernelGGL((k_rms_norm_grad<dt, st, gt, false, lpr, ch>), dim3((unsigned)a.rows), dim3(kGradThreads), 0, s, a);
    }); }); });
  });
  ANC_LAUNCH_CHECK();
  if (a.rows > 1) hipLaunchKernelGGL(k_gain_sum, dim3((unsigned)((H + 31) / 32)), dim3(kSumThreads), 0, s, (const float *)workspace, (float *)dgain, a.rows, (int)H, a.accumulate);
  ANC_LAUNCH_CHECK();
  return ANC_OK;
}
