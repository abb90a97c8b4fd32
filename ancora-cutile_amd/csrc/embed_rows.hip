// Input embedding on either side of the step: the lookup of its rows, and its gradient from ids grouped on the device
// (group.hip).
//     lookup:    out[i] = scale * table[ids[i]], a zero row where ids[i] names none
//     gradient:  dE[id] += scale * (sum of dy[i] over the positions i that hold id)
#include "rows.h"

namespace {

using namespace anc_rows;

// One piece of VEC elements per lane, (row, piece) flattened over the grid.
constexpr int kLookupLanes = 256;
template <int TT, int TO, int VEC>
__global__ void __launch_bounds__(kLookupLanes)
k_embed_lookup(const void *__restrict__ ids, int wide, int64_t n, int64_t V, uint32_t pieces, int64_t H, float scale,
               const elem_t<TT> *__restrict__ table, elem_t<TO> *__restrict__ out) {
  const int64_t i = (int64_t)blockIdx.x * kLookupLanes + threadIdx.x;
  const int64_t row = i / pieces;
  if (row >= n) return;
  const int64_t col = (i - row * pieces) * VEC;
  const int64_t id = wide ? ((const int64_t *)ids)[row] : (int64_t)((const int32_t *)ids)[row];
  float x[VEC];
  if (id >= 0 && id < V) {
    widen<TT, VEC>(load<TT, VEC>(table + id * H + col), x);
#pragma unroll
    for (int k = 0; k < VEC; ++k) x[k] = x[k] * scale;
  } else {
#pragma unroll
    for (int k = 0; k < VEC; ++k) x[k] = 0.0f;
  }
  store<TO, VEC>(out + row * H + col, x);
}

// The gradient walks the sorted positions in chunks of `chunk` (at most 64): a workgroup takes one chunk's rows of dy one after the
// other, and a group that lies inside the chunk is finished there. Of a group that reaches over an edge the chunk leaves a partial row,
// of the group that comes in (part 0) and of the one that goes out (part 1; a group that fills the chunk is part 0), and
// k_embed_dw_join adds them up in ascending order. Work is even whatever the ids: one id may hold most of the batch.
struct EmbedDw {
  const int32_t *srt, *start, *cnt, *key, *grp;
  int64_t n, V, H;
  int chunk;
  float scale;
  float *out, *compact, *part;
};
constexpr int kDwLanes = 256;

template <int VEC> __device__ __forceinline__ void put_row(const EmbedDw &p, int g, int64_t key, int64_t col, const float (&acc)[VEC]) {
  float x[VEC];
  if (p.compact != nullptr) {
#pragma unroll
    for (int k = 0; k < VEC; ++k) x[k] = p.scale * acc[k];
    store<ANC_F32, VEC>(p.compact + (int64_t)g * p.H + col, x);
  } else {
    float *at = p.out + key * p.H + col;
    widen<ANC_F32, VEC>(load<ANC_F32, VEC>(at), x);
#pragma unroll
    for (int k = 0; k < VEC; ++k) x[k] = x[k] + p.scale * acc[k];
    store<ANC_F32, VEC>(at, x);
  }
}

template <int TD, int VEC>
__global__ void __launch_bounds__(kDwLanes) k_embed_dw(EmbedDw p, const elem_t<TD> *__restrict__ dy) {
  const int lane = (int)(threadIdx.x & 63);
  const int64_t p0 = (int64_t)blockIdx.x * p.chunk, here = p0 + lane;
  const bool in = lane < p.chunk && here < p.n;
  const int idx = in ? p.srt[here] : 0, grp = in ? p.grp[here] : -1, key = in ? p.key[here] : 0;
  const int came = p0 > 0 ? p.grp[p0 - 1] : -1;                          // the group before the chunk
  const int goes = p0 + p.chunk < p.n ? p.grp[p0 + p.chunk] : -1;        // ... and behind it
  const int m = __popcll(__ballot(grp >= 0));                            // (ids that name no row lie at the end)
  const int64_t col = ((int64_t)blockIdx.y * blockDim.x + threadIdx.x) * VEC;
  const bool live = col < p.H;
  const int64_t c0 = live ? col : 0;                                     // (every lane stays: its indices serve the others)
  float acc[VEC];
  int cur = -1, cur_key = 0;
  auto flush = [&]() {
    if (cur < 0 || !live) return;
    if (cur == came || cur == goes)
      store<ANC_F32, VEC>(p.part + ((int64_t)blockIdx.x * 2 + (cur == came ? 0 : 1)) * p.H + c0, acc);
    else
      put_row<VEC>(p, cur, cur_key, c0, acc);
  };
  constexpr int D = 8;
  for (int i = 0; i < m; i += D) {
    Raw<TD, VEC> v[D];
#pragma unroll
    for (int j = 0; j < D; ++j) {
      const int r = __builtin_amdgcn_readlane(idx, i + j < m ? i + j : m - 1);
      v[j] = load<TD, VEC>(dy + (int64_t)r * p.H + c0);
    }
#pragma unroll
    for (int j = 0; j < D; ++j) {
      if (i + j >= m) break;
      const int g = __builtin_amdgcn_readlane(grp, i + j);
      if (g != cur) {
        flush();
        cur = g;
        cur_key = __builtin_amdgcn_readlane(key, i + j);
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[k] = 0.0f;
      }
      float x[VEC];
      widen<TD, VEC>(v[j], x);
#pragma unroll
      for (int k = 0; k < VEC; ++k) acc[k] = acc[k] + x[k];
    }
  }
  flush();
}

// Chunk c's part 1 begins a group that goes on: the parts of it, in order. The four wavefronts take a quarter of the list each
// (a third of 65536 positions on one id: 676 partial rows), their sums meet in LDS.
template <int VEC>
__global__ void __launch_bounds__(kDwLanes) k_embed_dw_join(EmbedDw p) {
  constexpr int W = kDwLanes / 64;
  __shared__ float sums[W][64 * VEC];
  const int64_t c = blockIdx.x, last = (c + 1) * p.chunk - 1;
  if (last + 1 >= p.n) return;
  const int g = p.grp[last];
  if (g < 0 || p.grp[last + 1] != g || (c > 0 && p.grp[last - p.chunk] == g)) return;     // (uniform over the workgroup)
  const int64_t ce = ((int64_t)p.start[g] + p.cnt[g] - 1) / p.chunk;
  const int lane = (int)(threadIdx.x & 63), wave = (int)(threadIdx.x >> 6);
  const int64_t col = ((int64_t)blockIdx.y * 64 + lane) * VEC;
  const bool live = col < p.H;
  const int64_t c0 = live ? col : 0, many = ce - c + 1, per = (many + W - 1) / W;
  const int64_t lo = wave * per < many ? wave * per : many, hi = lo + per < many ? lo + per : many;
  float acc[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) acc[k] = 0.0f;
  constexpr int D = 8;
  for (int64_t i = lo; i < hi; i += D) {
    Raw<ANC_F32, VEC> v[D];
#pragma unroll
    for (int j = 0; j < D; ++j) {
      const int64_t q = i + j < hi ? i + j : hi - 1;
      v[j] = load<ANC_F32, VEC>(p.part + ((c + q) * 2 + (q == 0 ? 1 : 0)) * p.H + c0);
    }
#pragma unroll
    for (int j = 0; j < D; ++j) {
      if (i + j >= hi) break;
      float x[VEC];
      widen<ANC_F32, VEC>(v[j], x);
#pragma unroll
      for (int k = 0; k < VEC; ++k) acc[k] = acc[k] + x[k];
    }
  }
#pragma unroll
  for (int k = 0; k < VEC; ++k) sums[wave][lane * VEC + k] = acc[k];
  __syncthreads();
  if (wave != 0 || !live) return;
#pragma unroll
  for (int w = 1; w < W; ++w)
#pragma unroll
    for (int k = 0; k < VEC; ++k) acc[k] = acc[k] + sums[w][lane * VEC + k];
  put_row<VEC>(p, g, p.key[last], c0, acc);
}

// Positions per chunk: enough chunks to fill the card, at most 64 (one index per lane).
constexpr int64_t kChunk16Most = 16384, kChunk32Most = 32768;
int dw_chunk(int64_t n) { return n <= kChunk16Most ? 16 : n <= kChunk32Most ? 32 : 64; }
int64_t dw_chunks(int64_t n) { return (n + dw_chunk(n) - 1) / dw_chunk(n); }
constexpr int64_t kMostPositions = 1ll << 20;

}  // namespace

extern "C" int anc_embed_lookup(uint64_t ids, int32_t ids_bytes, int64_t n, uint64_t table, int table_type, int64_t V, int64_t H,
                                float scale, uint64_t out, int out_type, uint64_t stream) {
  ANC_REQUIRE(n >= 0 && n < (1ll << 31) && V > 0 && V < (1ll << 40) && H > 0 && H <= (1ll << 20), "anc_embed_lookup: n=%lld, V=%lld, H=%lld",
              (long long)n, (long long)V, (long long)H);
  ANC_REQUIRE(ids_bytes == 4 || ids_bytes == 8, "anc_embed_lookup: ids of %d bytes (4 or 8)", (int)ids_bytes);
  ANC_REQUIRE(type_ok(table_type) && type_ok(out_type), "anc_embed_lookup: types %d and %d", table_type, out_type);
  if (n == 0) return ANC_OK;
  ANC_REQUIRE(ids && table && out, "anc_embed_lookup: null pointer");
  ANC_REQUIRE(ids % (uint64_t)ids_bytes == 0 && table % (uint64_t)elem_size(table_type) == 0 && out % (uint64_t)elem_size(out_type) == 0,
              "anc_embed_lookup: misaligned pointers");
  const Ptr ps[2] = {{table, table_type}, {out, out_type}};
  const int vec = piece(H, ps);
  const int64_t blocks = (n * (H / vec) + kLookupLanes - 1) / kLookupLanes;
  ANC_REQUIRE(blocks < (1ll << 31), "anc_embed_lookup: %lld rows of %lld are too many for one call", (long long)n, (long long)H);
  hipStream_t s = anc_stream(stream);
  AncProfScope prof(ANC_PROF_MISC, s);
  with_type(table_type, [&](auto tt) {
    with_type(out_type, [&](auto to) {
      with_piece(vec, [&](auto v) {
        constexpr int TT = decltype(tt)::value, TO = decltype(to)::value, VEC = decltype(v)::value;
        hipLaunchKernelGGL((k_embed_lookup<TT, TO, VEC>), dim3((unsigned)blocks), dim3(kLookupLanes), 0, s, (const void *)ids,
                           ids_bytes == 8, n, V, (uint32_t)(H / VEC), H, scale, (const elem_t<TT> *)table, (elem_t<TO> *)out);
      });
    });
  });
  ANC_LAUNCH_CHECK();
  return ANC_OK;
}

// Enough for every batch of up to M positions.
extern "C" int64_t anc_embed_dw_workspace_bytes(int64_t M, int64_t H) {
  if (M <= 0 || M > kMostPositions || H <= 0 || H > (1ll << 20)) {
    anc_set_error("anc_embed_dw_workspace_bytes: M=%lld (1 .. %lld), H=%lld", (long long)M, (long long)kMostPositions, (long long)H);
    return -1;
  }
  int64_t most = dw_chunks(M);
  for (int64_t edge : {kChunk16Most, kChunk32Most})
    if (edge < M && dw_chunks(edge) > most) most = dw_chunks(edge);
  return most * 2 * H * 4;
}

extern "C" int anc_embed_dw(uint64_t srt, uint64_t start, uint64_t cnt, uint64_t key, uint64_t grp, int64_t n, uint64_t dy, int dy_type,
                            int64_t H, float scale, uint64_t out, uint64_t compact, int64_t V, uint64_t workspace,
                            int64_t workspace_bytes, uint64_t stream) {
  ANC_REQUIRE(n >= 0 && n <= kMostPositions && H > 0 && H <= (1ll << 20) && (out == 0 || V > 0), "anc_embed_dw: n=%lld (at most %lld), V=%lld, H=%lld",
              (long long)n, (long long)kMostPositions, (long long)V, (long long)H);
  ANC_REQUIRE(type_ok(dy_type), "anc_embed_dw: type %d", dy_type);
  ANC_REQUIRE((out != 0) != (compact != 0), "anc_embed_dw: one of out and compact");
  if (n == 0) return ANC_OK;
  ANC_REQUIRE(srt && start && cnt && key && grp && dy && workspace, "anc_embed_dw: null pointer");
  ANC_REQUIRE(((srt | start | cnt | key | grp | out | compact) & 3) == 0 && dy % (uint64_t)elem_size(dy_type) == 0 && (workspace & 15) == 0,
              "anc_embed_dw: misaligned pointers");
  const int64_t chunks = dw_chunks(n), need = chunks * 2 * H * 4;
  ANC_REQUIRE(workspace_bytes >= need, "anc_embed_dw: workspace holds %lld bytes, %lld needed", (long long)workspace_bytes, (long long)need);
  const Ptr ps[2] = {{dy, dy_type}, {out | compact, ANC_F32}};
  const int vec = piece(H, ps);
  hipStream_t s = anc_stream(stream);
  AncProfScope prof(ANC_PROF_MISC, s);
  EmbedDw p{(const int32_t *)srt, (const int32_t *)start, (const int32_t *)cnt, (const int32_t *)key, (const int32_t *)grp,
            n, V, H, dw_chunk(n), scale, (float *)out, (float *)compact, (float *)workspace};
  with_piece(vec, [&](auto v) {
    constexpr int VEC = decltype(v)::value;
    const int64_t waves = (H + 64 * VEC - 1) / (64 * VEC), wide = waves < kDwLanes / 64 ? waves : kDwLanes / 64;
    with_type(dy_type, [&](auto t) {
      constexpr int T = decltype(t)::value;
      hipLaunchKernelGGL((k_embed_dw<T, VEC>), dim3((unsigned)chunks, (unsigned)((waves + wide - 1) / wide)), dim3((unsigned)(64 * wide)), 0,
                         s, p, (const elem_t<T> *)dy);
    });
    if (chunks > 1)
      hipLaunchKernelGGL((k_embed_dw_join<VEC>), dim3((unsigned)(chunks - 1), (unsigned)waves), dim3(kDwLanes), 0, s, p);
  });
  ANC_LAUNCH_CHECK();
  return ANC_OK;
}
