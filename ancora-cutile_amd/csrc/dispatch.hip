// Rows of tokens to the experts' segments and back, over the slots that anc_route (group.hip) assigned: slot[t * k + j] is
// the place of token t's choice j, -1 where the choice names no expert (a masked token).
//     dispatch:      xs[slot] = x[t]; the rows that fill up a segment become zero
//     combine:       y[t] = sum over j of w[t, j] * ys[slot]          (w = 1: the gradient of dispatch)
//     combine_grad:  dys[slot] = w[t, j] * dy[t];  dw[t, j] = <dy[t], ys[slot]>
// All are bound by memory. They go by token, not by slot: a token's own row is read or written once for its k choices. A slot outside
// [0, capacity) is taken for none, whatever the array holds.
// Measured: 8192 tokens of 2 choices, rows of 1024 bf16 values: dispatch 9.9 us, its gradient 9.8, combine into fp32 rows 11.4 (5.6 TB/s);
// combine_grad of 16384 tokens of 8 choices, rows of 640: 66 us, 5.2 TB/s (a large copy: 5.9).
#include "rows.h"

namespace {

using namespace anc_rows;

constexpr int kLanes = 256;
constexpr int kPadRows = 8;                 // rows that one workgroup clears

__device__ __forceinline__ int64_t in_range(int64_t slot, int64_t capacity) { return slot < capacity ? slot : -1; }

// Rows between an expert's last token and the end of its segment: workgroup `b` of those that clear them.
template <int T, int VEC, bool TAIL>
__device__ __forceinline__ void clear_padding(int b, int align, const int32_t *counts, const int32_t *offsets, int64_t capacity, int64_t H,
                                              elem_t<T> *out) {
  const int per = (align - 1 + kPadRows - 1) / kPadRows, e = b / per;
  const int64_t from = (int64_t)offsets[e] + counts[e] + (int64_t)(b - e * per) * kPadRows, last = offsets[e + 1];
  const int64_t end = last < capacity ? last : capacity;
  const int64_t to = from + kPadRows < end ? from + kPadRows : end;
  if (from < 0 || from >= to) return;
  float zero[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) zero[k] = 0.0f;
  const Raw<T, VEC> r = narrow<T, VEC>(zero);        // (the rows lie behind each other: one long row)
  for (int64_t i = threadIdx.x * VEC; i < (to - from) * H; i += kLanes * VEC) store<T, VEC, TAIL>(out + from * H, r, piece_at<VEC, TAIL>(i, (to - from) * H));
}

template <int T, bool TAIL>
__global__ void __launch_bounds__(kLanes)
k_dispatch(const int32_t *__restrict__ slot, const int32_t *__restrict__ counts, const int32_t *__restrict__ offsets, uint32_t total,
           int k, int align, uint32_t main_blocks, FastDiv pieces, int64_t capacity, int64_t H, const elem_t<T> *__restrict__ x,
           elem_t<T> *__restrict__ xs) {
  constexpr int VEC = piece_of<T, T>;
  if (blockIdx.x >= main_blocks) {
    clear_padding<T, VEC, TAIL>((int)(blockIdx.x - main_blocks), align, counts, offsets, capacity, H, xs);
    return;
  }
  const uint32_t i = blockIdx.x * (uint32_t)kLanes + threadIdx.x;
  if (i >= total) return;
  const uint32_t t = pieces.div(i);
  const Piece c = piece_at<VEC, TAIL>((int64_t)(i - t * pieces.d) * VEC, H);
  const Raw<T, VEC> v = load<T, VEC, TAIL>(x + (int64_t)t * H, c);
  const int32_t *to = slot + (int64_t)t * k;
  constexpr int D = 4;
  for (int j0 = 0; j0 < k; j0 += D) {
    int64_t s[D];
#pragma unroll
    for (int j = 0; j < D; ++j) s[j] = in_range(to[j0 + j < k ? j0 + j : k - 1], capacity);
#pragma unroll
    for (int j = 0; j < D; ++j)
      if (j0 + j < k && s[j] >= 0) store<T, VEC, TAIL>(xs + s[j] * H, v, c);
  }
}

template <int TI, int TO, bool TAIL, bool WEIGHTS>
__global__ void __launch_bounds__(kLanes)
k_combine(const int32_t *__restrict__ slot, const float *__restrict__ w, uint32_t total, int k, FastDiv pieces, int64_t capacity, int64_t H,
          const elem_t<TI> *__restrict__ ys, elem_t<TO> *__restrict__ y) {
  constexpr int VEC = piece_of<TI, TO>;
  const uint32_t i = blockIdx.x * (uint32_t)kLanes + threadIdx.x;
  if (i >= total) return;
  const uint32_t row = pieces.div(i);
  const int64_t t = row;
  const Piece c = piece_at<VEC, TAIL>((int64_t)(i - row * pieces.d) * VEC, H);
  float acc[VEC];
#pragma unroll
  for (int q = 0; q < VEC; ++q) acc[q] = 0.0f;
  constexpr int D = 4;
  for (int j0 = 0; j0 < k; j0 += D) {
    Raw<TI, VEC> v[D];
    int64_t s[D];
    float f[D];
#pragma unroll
    for (int j = 0; j < D; ++j) {
      const int64_t a = t * k + (j0 + j < k ? j0 + j : k - 1);
      const int64_t at = in_range(slot[a], capacity);
      f[j] = WEIGHTS ? w[a] : 1.0f;
      s[j] = j0 + j < k ? at : -1;
    }
#pragma unroll
    for (int j = 0; j < D; ++j)
      if (s[j] >= 0) v[j] = load<TI, VEC, TAIL>(ys + s[j] * H, c);
#pragma unroll
    for (int j = 0; j < D; ++j) {
      if (s[j] < 0) continue;
      float a[VEC];
      widen<TI, VEC>(v[j], a);
#pragma unroll
      for (int q = 0; q < VEC; ++q) acc[q] = WEIGHTS ? fmaf(f[j], a[q], acc[q]) : acc[q] + a[q];
    }
  }
  store<TO, VEC, TAIL>(y + t * H, narrow<TO, VEC>(acc), c);
}

// One wavefront per token, four choices at a time: their rows are in flight together, dy comes from the caches for the next
// four. The four products' sums over the lanes are made together: at the first two steps of the butterfly a lane hands half of its sums
// on and keeps the other half, so that four sums take 7 exchanges instead of 24.
template <int TY, int TS, bool TAIL, bool ONCE>
__global__ void __launch_bounds__(kLanes)
k_combine_grad(const int32_t *__restrict__ slot, const float *__restrict__ w, const int32_t *__restrict__ counts,
               const int32_t *__restrict__ offsets, int64_t tokens, int k, int align, int64_t main_blocks, int64_t capacity, int64_t H,
               const elem_t<TY> *__restrict__ dy, const elem_t<TS> *__restrict__ ys, elem_t<TS> *__restrict__ dys,
               float *__restrict__ dw) {
  constexpr int VEC = piece_of<TY, TS>;
  if ((int64_t)blockIdx.x >= main_blocks) {
    clear_padding<TS, VEC, TAIL>((int)((int64_t)blockIdx.x - main_blocks), align, counts, offsets, capacity, H, dys);
    return;
  }
  const int lane = (int)(threadIdx.x & 63);
  const int64_t t = (int64_t)blockIdx.x * (kLanes / 64) + __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  if (t >= tokens) return;
  constexpr int D = 4;
  for (int j0 = 0; j0 < k; j0 += D) {
    int64_t s[D];
    float f[D], dot[D];
#pragma unroll
    for (int j = 0; j < D; ++j) {
      const int64_t a = t * k + (j0 + j < k ? j0 + j : k - 1);
      s[j] = in_range(slot[a], capacity);
      f[j] = w[a];
      dot[j] = 0.0f;
      if (j0 + j >= k) s[j] = -1;
    }
    for (int64_t col = (int64_t)lane * VEC; col < H; col += 64 * VEC) {
      float g[VEC];
      Raw<TS, VEC> v[D];
      const Piece c = piece_at<VEC, TAIL>(col, H);
      const Raw<TY, VEC> own = load<TY, VEC, TAIL>(dy + t * H, c);
#pragma unroll
      for (int j = 0; j < D; ++j)
        if (s[j] >= 0) v[j] = load<TS, VEC, TAIL, ONCE>(ys + s[j] * H, c);
      widen<TY, VEC>(own, g);
#pragma unroll
      for (int j = 0; j < D; ++j) {
        if (s[j] < 0) continue;
        float a[VEC], o[VEC];
        widen<TS, VEC>(v[j], a);
#pragma unroll
        for (int q = 0; q < VEC; ++q) {
          if (!TAIL || q >= c.first) dot[j] = fmaf(g[q], a[q], dot[j]);
          o[q] = f[j] * g[q];
        }
        store<TS, VEC, TAIL, ONCE>(dys + s[j] * H, narrow<TS, VEC>(o), c);
      }
    }
    // lane bit 5 chooses the pair (0, 1) or (2, 3), bit 4 the one of the pair
    const bool hi = (lane & 32) != 0, odd = (lane & 16) != 0;
    const float a = (hi ? dot[2] : dot[0]) + __shfl_xor(hi ? dot[0] : dot[2], 32, 64);
    const float b = (hi ? dot[3] : dot[1]) + __shfl_xor(hi ? dot[1] : dot[3], 32, 64);
    float sum = (odd ? b : a) + __shfl_xor(odd ? a : b, 16, 64);
#pragma unroll
    for (int o = 8; o >= 1; o >>= 1) sum += __shfl_xor(sum, o, 64);
    const int j = j0 + (hi ? 2 : 0) + (odd ? 1 : 0);
    if ((lane & 15) == 0 && j < k) dw[t * k + j] = sum;
  }
}

int check_rows(const char *who, uint64_t slot, int64_t tokens, int64_t k, int64_t capacity, int64_t H) {
  ANC_REQUIRE(tokens >= 0 && tokens < (1ll << 31) && k > 0 && k <= 512 && H > 0 && H <= (1ll << 20) && tokens * k <= (1ll << 22),
              "%s: %lld tokens of width %lld with %lld choices", who, (long long)tokens, (long long)H, (long long)k);
  ANC_REQUIRE(slot != 0 && (slot & 3) == 0, "%s: null or misaligned slots", who);
  ANC_REQUIRE(capacity > 0 && capacity < (1ll << 31), "%s: room for %lld slots", who, (long long)capacity);
  return ANC_OK;
}
int check_segments(const char *who, uint64_t counts, uint64_t offsets, int64_t experts, int64_t align) {
  ANC_REQUIRE(counts && offsets && ((counts | offsets) & 3) == 0 && experts > 0 && experts <= 512 && align > 0 && align <= 256,
              "%s: bad segments (%lld experts, align %lld)", who, (long long)experts, (long long)align);
  return ANC_OK;
}
int64_t pad_blocks(int64_t experts, int64_t align) { return experts * ((align - 1 + kPadRows - 1) / kPadRows); }

}  // namespace

extern "C" int anc_dispatch(uint64_t slot, uint64_t counts, uint64_t offsets, int64_t tokens, int64_t k, int64_t experts, int64_t align,
                            uint64_t x, uint64_t xs, int64_t capacity, int type, int64_t H, uint64_t stream) {
  if (int rc = check_rows("anc_dispatch", slot, tokens, k, capacity, H)) return rc;
  if (int rc = check_segments("anc_dispatch", counts, offsets, experts, align)) return rc;
  ANC_REQUIRE(type_ok(type), "anc_dispatch: type %d", type);
  ANC_REQUIRE(x && xs && (x | xs) % (uint64_t)elem_size(type) == 0, "anc_dispatch: null or misaligned pointers");
  ANC_REQUIRE(anc_outputs_apart({{xs, capacity * H * elem_size(type)}, {x, tokens * H * elem_size(type)}, {slot, 4 * tokens * k}, {counts, 4 * experts},
                                 {offsets, 4 * experts + 4}}, 1),
              "anc_dispatch: xs overlaps an input");
  const int64_t vec = type == ANC_F32 ? 4 : 8, per_row = pieces_of(H, vec), most = kMostPieces / per_row;
  hipStream_t s = anc_stream(stream);
  AncProfScope prof(ANC_PROF_MISC, s);
  for (int64_t r = 0; r < tokens; r += most) {       // (the first launch clears the padding)
    const int64_t rows = tokens - r < most ? tokens - r : most, total = rows * per_row;
    const int64_t blocks = (total + kLanes - 1) / kLanes, all = blocks + (r == 0 ? pad_blocks(experts, align) : 0);
    with_type(type, [&](auto t) {
      with_flag(H % vec != 0, [&](auto tail) {
        constexpr int T = decltype(t)::value;
        hipLaunchKernelGGL((k_dispatch<T, decltype(tail)::value != 0>), dim3((unsigned)all), dim3(kLanes), 0, s, (const int32_t *)slot + r * k,
                           (const int32_t *)counts, (const int32_t *)offsets, (uint32_t)total, (int)k, (int)align, (uint32_t)blocks,
                           fast_div((uint32_t)per_row), capacity, H, (const elem_t<T> *)x + r * H, (elem_t<T> *)xs);
      });
    });
  }
  ANC_LAUNCH_CHECK();
  return ANC_OK;
}

extern "C" int anc_combine(uint64_t slot, uint64_t weights, int64_t tokens, int64_t k, uint64_t ys, int64_t capacity, int ys_type, uint64_t y, int y_type,
                           int64_t H, uint64_t stream) {
  if (int rc = check_rows("anc_combine", slot, tokens, k, capacity, H)) return rc;
  ANC_REQUIRE(type_ok(ys_type) && type_ok(y_type), "anc_combine: types %d and %d", ys_type, y_type);
  ANC_REQUIRE(ys && y && ys % (uint64_t)elem_size(ys_type) == 0 && y % (uint64_t)elem_size(y_type) == 0 && (weights & 3) == 0,
              "anc_combine: null or misaligned pointers");
  ANC_REQUIRE(anc_outputs_apart({{y, tokens * H * elem_size(y_type)}, {ys, capacity * H * elem_size(ys_type)}, {weights, weights != 0 ? 4 * tokens * k : 0},
                                 {slot, 4 * tokens * k}}, 1),
              "anc_combine: y overlaps an input");
  const int64_t vec = ys_type == ANC_F32 || y_type == ANC_F32 ? 4 : 8, per_row = pieces_of(H, vec), most = kMostPieces / per_row;
  hipStream_t s = anc_stream(stream);
  AncProfScope prof(ANC_PROF_MISC, s);
  for (int64_t r = 0; r < tokens; r += most) {
    const int64_t rows = tokens - r < most ? tokens - r : most, total = rows * per_row;
    with_type(ys_type, [&](auto ti) {
      with_type(y_type, [&](auto to) {
        with_flag(H % vec != 0, [&](auto tail) {
          constexpr int TI = decltype(ti)::value, TO = decltype(to)::value;
          constexpr bool TAIL = decltype(tail)::value != 0;
          auto kernel = weights != 0 ? k_combine<TI, TO, TAIL, true> : k_combine<TI, TO, TAIL, false>;
          hipLaunchKernelGGL(kernel, dim3((unsigned)((total + kLanes - 1) / kLanes)), dim3(kLanes), 0, s, (const int32_t *)slot + r * k,
                             weights != 0 ? (const float *)weights + r * k : (const float *)nullptr, (uint32_t)total, (int)k,
                             fast_div((uint32_t)per_row), capacity, H, (const elem_t<TI> *)ys, (elem_t<TO> *)y + r * H);
        });
      });
    });
  }
  ANC_LAUNCH_CHECK();
  return ANC_OK;
}

extern "C" int anc_combine_grad(uint64_t slot, uint64_t weights, uint64_t counts, uint64_t offsets, int64_t tokens, int64_t k,
                                int64_t experts, int64_t align, uint64_t dy, int dy_type, uint64_t ys, uint64_t dys, int64_t capacity,
                                int ys_type, uint64_t dw, int64_t H, uint64_t stream) {
  if (int rc = check_rows("anc_combine_grad", slot, tokens, k, capacity, H)) return rc;
  if (int rc = check_segments("anc_combine_grad", counts, offsets, experts, align)) return rc;
  ANC_REQUIRE(type_ok(dy_type) && type_ok(ys_type), "anc_combine_grad: types %d and %d", dy_type, ys_type);
  ANC_REQUIRE(weights && dy && ys && dys && dw && ((weights | dw) & 3) == 0 && dy % (uint64_t)elem_size(dy_type) == 0 &&
                  (ys | dys) % (uint64_t)elem_size(ys_type) == 0,
              "anc_combine_grad: null or misaligned pointers");
  const int64_t dy_bytes = tokens * H * elem_size(dy_type), ys_bytes = capacity * H * elem_size(ys_type), w_bytes = tokens * k * 4;
  ANC_REQUIRE(anc_outputs_apart({{dys, ys_bytes}, {dw, w_bytes}, {ys, ys_bytes}, {dy, dy_bytes}, {weights, w_bytes}, {slot, w_bytes}, {counts, 4 * experts},
                                 {offsets, 4 * experts + 4}}, 2),
              "anc_combine_grad: an output overlaps another buffer");
  const int64_t vec = dy_type == ANC_F32 || ys_type == ANC_F32 ? 4 : 8;
  const int64_t blocks = (tokens + kLanes / 64 - 1) / (kLanes / 64), all = blocks + pad_blocks(experts, align);
  if (tokens == 0) return ANC_OK;
  hipStream_t s = anc_stream(stream);
  AncProfScope prof(ANC_PROF_MISC, s);
  with_type(dy_type, [&](auto ty) {
    with_type(ys_type, [&](auto ts) {
      with_flag(H % vec != 0, [&](auto tail) {
        constexpr int TY = decltype(ty)::value, TS = decltype(ts)::value;
        constexpr bool TAIL = decltype(tail)::value != 0;
        const bool once = tokens * k * H * elem_size(ys_type) > kCached;
        auto kernel = once ? k_combine_grad<TY, TS, TAIL, true> : k_combine_grad<TY, TS, TAIL, false>;
        hipLaunchKernelGGL(kernel, dim3((unsigned)all), dim3(kLanes), 0, s, (const int32_t *)slot,
                           (const float *)weights, (const int32_t *)counts, (const int32_t *)offsets, tokens, (int)k, (int)align, blocks, capacity, H,
                           (const elem_t<TY> *)dy, (const elem_t<TS> *)ys, (elem_t<TS> *)dys, (float *)dw);
      });
    });
  });
  ANC_LAUNCH_CHECK();
  return ANC_OK;
}
