// Input embedding on either side of the step: the lookup of its rows, and its gradient from ids grouped on the device
// (group.hip).
//     lookup:    out[i] = scale * table[ids[i]], a zero row where ids[i] names none
//     gradient:  dE[id] += scale * (sum of dy[i] over the positions i that hold id)
#include "rows.h"

namespace {

using namespace anc_rows;

// U pieces of VEC elements per lane, (row, piece) flattened over the grid. The U ids and then the U pieces are in flight together.
constexpr int kLookupLanes = 256;
template <int TT, int TO, bool TAIL, int U, bool ONCE>
__global__ void __launch_bounds__(kLookupLanes)
k_embed_lookup(const void *__restrict__ ids, int wide, uint32_t total, int64_t V, FastDiv pieces, int64_t H, float scale,
               const elem_t<TT> *__restrict__ table, elem_t<TO> *__restrict__ out) {
  constexpr int VEC = piece_of<TT, TO>;
  const uint32_t first = blockIdx.x * (uint32_t)(kLookupLanes * U) + threadIdx.x;
  uint32_t row[U];
  int64_t id[U];
  Piece c[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t i = first + u * kLookupLanes < total ? first + u * kLookupLanes : total - 1;
    row[u] = pieces.div(i);
    c[u] = piece_at<VEC, TAIL>((int64_t)(i - row[u] * pieces.d) * VEC, H);
    id[u] = wide ? ((const int64_t *)ids)[row[u]] : (int64_t)((const int32_t *)ids)[row[u]];
  }
  Raw<TT, VEC> r[U];
#pragma unroll
  for (int u = 0; u < U; ++u) r[u] = load<TT, VEC, TAIL>(table + (id[u] >= 0 && id[u] < V ? id[u] : 0) * H, c[u]);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (first + u * kLookupLanes >= total) return;
    float x[VEC];
    widen<TT, VEC>(r[u], x);
    const bool there = id[u] >= 0 && id[u] < V;
#pragma unroll
    for (int k = 0; k < VEC; ++k) x[k] = there ? x[k] * scale : 0.0f;
    store<TO, VEC, TAIL, ONCE>(out + (int64_t)row[u] * H, narrow<TO, VEC>(x), c[u]);
  }
}

// The gradient walks the sorted positions in chunks: a workgroup of SUBS teams, each of which adds up the rows of dy of `sub` (at most 64)
// positions one after the other. A group that lies inside a team's positions is finished there. Of one that reaches over an edge the team
// leaves a row in LDS, of the group that comes in (head) and of the one that begins and goes out (tail), and the teams put
// together what meets inside the chunk. What reaches over the chunk's edges goes to memory the same way, part 0 of the group that comes in and
// part 1 of the one that begins and goes out, and k_embed_dw_join adds those up in ascending order. Work is even whatever the ids: one
// id may hold most of the batch.
struct EmbedDw {
  const int32_t *srt, *start, *cnt, *key, *grp;
  int64_t n, V, H, pitch;                            // pitch: between rows of part, whole pieces
  int sub, chunk;                                    // positions of a team, of a workgroup
  float scale;
  float *out, *compact, *part;
};
constexpr int kSubs = 4, kFewSubs = 16;              // teams; of the one workgroup that few positions make
constexpr int kDwLanes = 256;                        // most lanes of a team, and of the join

template <int VEC, bool TAIL, bool DENSE>
__device__ __forceinline__ void put_row(const EmbedDw &p, int64_t row, const Piece &c, const float (&acc)[VEC]) {
  float x[VEC];
  float *to = (DENSE ? p.out : p.compact) + row * p.H;
  if constexpr (DENSE) widen<ANC_F32, VEC>(load<ANC_F32, VEC, TAIL>(to, c), x);
#pragma unroll
  for (int k = 0; k < VEC; ++k) x[k] = DENSE ? x[k] + p.scale * acc[k] : p.scale * acc[k];
  store<ANC_F32, VEC, TAIL, false, DENSE>(to, narrow<ANC_F32, VEC>(x), c);
}

template <int TD, bool TAIL, bool DENSE, bool ONCE, int SUBS>
__global__ void __launch_bounds__(kDwLanes * kSubs) k_embed_dw(EmbedDw p, const elem_t<TD> *__restrict__ dy) {
  constexpr int VEC = piece_of<TD, TD>;
  extern __shared__ __attribute__((aligned(16))) float edge[];                    // [SUBS][head, tail][lanes * VEC]
  __shared__ int flags[SUBS];                       // 1: a head, 2: its group goes out again, 4: a tail
  const int lane = (int)(threadIdx.x & 63), team = __builtin_amdgcn_readfirstlane((int)threadIdx.y);
  const int64_t p0 = (int64_t)blockIdx.x * p.chunk + (int64_t)team * p.sub, here = p0 + lane;
  const bool in = lane < p.sub && here < p.n;
  const int64_t at = in ? here : p.n - 1;
  const int row = p.srt[at], key = p.key[at], read = p.grp[at], idx = (uint32_t)row < (uint32_t)p.n ? row : 0;
  const int grp = in && (uint32_t)read < (uint32_t)p.n && (uint32_t)key < (uint64_t)p.V ? read : -1;      // (whatever the arrays hold, no other row is touched)
  const int came = p0 > 0 && p0 < p.n ? p.grp[p0 - 1] : -1;              // the group before the team's positions
  const int goes = p0 + p.sub < p.n ? p.grp[p0 + p.sub] : -1;            // ... and behind them
  const int m = __popcll(__ballot(grp >= 0));                            // (ids that name no row lie at the end)
  const int64_t col = ((int64_t)blockIdx.y * blockDim.x + threadIdx.x) * VEC;
  const bool live = col < p.H;
  const Piece c = piece_at<VEC, TAIL>(live ? col : 0, p.H);              // (every lane stays: its indices serve the others)
  const int width = (int)blockDim.x * VEC;
  float *head = edge + team * 2 * width + threadIdx.x * VEC, *tail = head + width;
  float acc[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) acc[k] = 0.0f;
  int state = 0, tail_grp = -1, tail_key = 0;
  constexpr int D = DENSE ? 4 : 8;
  for (int i = 0; i < m; i += D) {
    Raw<TD, VEC> v[D];
    Raw<ANC_F32, VEC> old[DENSE ? D : 1];
    int g[D], next[D];
#pragma unroll
    for (int j = 0; j < D; ++j) {
      const int q = i + j < m ? i + j : m - 1;
      g[j] = __builtin_amdgcn_readlane(grp, q);
      next[j] = q + 1 < m ? __builtin_amdgcn_readlane(grp, q + 1) : -1;  // (a group that goes on behind ends here, too)
      v[j] = load<TD, VEC, TAIL, ONCE>(dy + (int64_t)__builtin_amdgcn_readlane(idx, q) * p.H, c);
      if constexpr (DENSE)
        if (next[j] != g[j] && g[j] != came && g[j] != goes && g[j] >= 0)
          old[j] = load<ANC_F32, VEC, TAIL>(p.out + (int64_t)__builtin_amdgcn_readlane(key, q) * p.H, c);
    }
#pragma unroll
    for (int j = 0; j < D; ++j) {
      if (i + j >= m) continue;
      float x[VEC];
      widen<TD, VEC>(v[j], x);
#pragma unroll
      for (int k = 0; k < VEC; ++k) acc[k] = acc[k] + x[k];
      if (next[j] == g[j]) continue;
      if (g[j] < 0) {                                // (arrays out of order only)
      } else if (g[j] == came) {
        state |= g[j] == goes ? 3 : 1;
        *(Raw<ANC_F32, VEC> *)head = narrow<ANC_F32, VEC>(acc);
      } else if (g[j] == goes) {
        state |= 4;
        tail_grp = g[j];
        tail_key = __builtin_amdgcn_readlane(key, i + j);
        *(Raw<ANC_F32, VEC> *)tail = narrow<ANC_F32, VEC>(acc);
      } else if (live) {
        if constexpr (DENSE) widen<ANC_F32, VEC>(old[j], x);
#pragma unroll
        for (int k = 0; k < VEC; ++k) x[k] = DENSE ? x[k] + p.scale * acc[k] : p.scale * acc[k];
        float *to = DENSE ? p.out + (int64_t)__builtin_amdgcn_readlane(key, i + j) * p.H : p.compact + (int64_t)g[j] * p.H;
        store<ANC_F32, VEC, TAIL, false, DENSE>(to, narrow<ANC_F32, VEC>(x), c);
      }
#pragma unroll
      for (int k = 0; k < VEC; ++k) acc[k] = 0.0f;
    }
  }
  if (threadIdx.x == 0) flags[team] = state;
  __syncthreads();
  auto add_head = [&](int t) {
    float x[VEC];
    widen<ANC_F32, VEC>(*(const Raw<ANC_F32, VEC> *)(edge + t * 2 * width + threadIdx.x * VEC), x);
#pragma unroll
    for (int k = 0; k < VEC; ++k) acc[k] = acc[k] + x[k];
  };
  if (state & 4) {                                   // what begins here and goes on
    widen<ANC_F32, VEC>(*(const Raw<ANC_F32, VEC> *)tail, acc);
    int t = team + 1;
    for (; t < SUBS; ++t) {
      add_head(t);
      if (!(flags[t] & 2)) break;
    }
    if (live) {
      if (t < SUBS) put_row<VEC, TAIL, DENSE>(p, DENSE ? (int64_t)tail_key : (int64_t)tail_grp, c, acc);
      else store<ANC_F32, VEC, TAIL>(p.part + ((int64_t)blockIdx.x * 2 + 1) * p.pitch, narrow<ANC_F32, VEC>(acc), c);
    }
  }
  if (team == 0 && (state & 1)) {                    // what came into the chunk
#pragma unroll
    for (int k = 0; k < VEC; ++k) acc[k] = 0.0f;
    for (int t = 0; t < SUBS; ++t) {
      add_head(t);
      if (!(flags[t] & 2)) break;
    }
    if (live) store<ANC_F32, VEC, TAIL>(p.part + (int64_t)blockIdx.x * 2 * p.pitch, narrow<ANC_F32, VEC>(acc), c);
  }
}

// Chunk c's part 1 begins a group that goes on: the parts of it, in order. The four wavefronts take a quarter of the list each
// (a third of 65536 positions on one id: 85 rows), 8 rows in flight, and their sums meet in LDS.
template <bool TAIL>
__global__ void __launch_bounds__(kDwLanes) k_embed_dw_join(EmbedDw p) {
  constexpr int W = kDwLanes / 64, VEC = 4;           // (narrow pieces: more wavefronts on a long list)
  __shared__ float sums[W][64 * VEC];
  const int64_t c = blockIdx.x, last = (c + 1) * p.chunk - 1;
  if (last + 1 >= p.n) return;
  const int g = p.grp[last], behind = p.grp[last + 1], before = c > 0 ? p.grp[last - p.chunk] : -1;
  if ((uint32_t)g >= (uint32_t)p.n || behind != g || before == g) return;     // (uniform over the workgroup)
  const int64_t key = p.key[last], end = (int64_t)p.start[g] + p.cnt[g], ce = ((end < p.n ? end : p.n) - 1) / p.chunk;
  if (ce < c || key < 0 || key >= p.V) return;
  const int lane = (int)(threadIdx.x & 63), wave = (int)(threadIdx.x >> 6);
  const int64_t col = ((int64_t)blockIdx.y * 64 + lane) * VEC;
  const bool live = col < p.H;
  const Piece pc = piece_at<VEC, TAIL>(live ? col : 0, p.H);
  const int64_t many = ce - c + 1, per = (many + W - 1) / W;
  const int64_t lo = wave * per < many ? wave * per : many, hi = lo + per < many ? lo + per : many;
  float *to = p.compact != nullptr ? p.compact + (int64_t)g * p.H : p.out + key * p.H;
  Raw<ANC_F32, VEC> old;
  if (p.compact == nullptr) old = load<ANC_F32, VEC, TAIL>(to, pc);
  float acc[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) acc[k] = 0.0f;
  constexpr int D = 8;
  for (int64_t i = lo; i < hi; i += D) {
    Raw<ANC_F32, VEC> v[D];
#pragma unroll
    for (int j = 0; j < D; ++j) {
      const int64_t q = i + j < hi ? i + j : hi - 1;
      v[j] = load<ANC_F32, VEC, TAIL>(p.part + ((c + q) * 2 + (q == 0 ? 1 : 0)) * p.pitch, pc);
    }
#pragma unroll
    for (int j = 0; j < D; ++j) {
      float x[VEC];
      widen<ANC_F32, VEC>(v[j], x);
      if (i + j < hi) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[k] = acc[k] + x[k];
      }
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
  float x[VEC];
  if (p.compact == nullptr) widen<ANC_F32, VEC>(old, x);
#pragma unroll
  for (int k = 0; k < VEC; ++k) x[k] = p.compact == nullptr ? x[k] + p.scale * acc[k] : p.scale * acc[k];
  store<ANC_F32, VEC, TAIL, false, true>(to, narrow<ANC_F32, VEC>(x), pc);
}

// Positions per team: enough chunks to fill the card while there are few, fewer partial rows where there are many. By n alone, so that the bits
// do not hang on the width. Gradient and join, us, mostly distinct ids, bf16 rows of 256, 1024 and 2048 values:
//   runs of 8 and 16:   8192 positions 7.9 and 9.9, 16.2 and 20.0, 29 and 27; 12288 8.9 and 10.3, 24.8 and 22.8, 38 and 43; 16384 10.2 and 11.4, 26.7 and
//                       26.0, 50 and 49
//   runs of 16 and 64:  32768 16.0 and 29.7, 44 and 63, 85 and 79; 65536 24.7 and 34.3, 71 and 74, 163 and 154; with a third of the positions on one id
//                       32768 17 and 28, 37 and 45, 72 and 67; 65536 28 and 33, 62 and 66, 151 and 147 (64 is right for wide rows only)
// Up to kFewMost all are one workgroup's, for 64 pieces of the rows each, and nothing is left to join (77 rows into a dense gradient 6.7 us, by
// the join 8.8; 128 rows 9.1 and 8.9, into compact rows 7.1 and 8.8; 200 rows, 16 to a team, 12.2 and 9.0).
constexpr int64_t kFewMost = kFewSubs * 8, kSub8Most = 8192, kSub16Most = 32768;
int dw_sub(int64_t n) { return n <= kFewSubs * 4 ? 4 : n <= kSub8Most ? 8 : n <= kSub16Most ? 16 : 64; }
int dw_chunk(int64_t n) { return (n <= kFewMost ? kFewSubs : kSubs) * dw_sub(n); }
int64_t dw_chunks(int64_t n) { return (n + dw_chunk(n) - 1) / dw_chunk(n); }
int64_t dw_pitch(int64_t H) { return (H + 7) / 8 * 8; }
constexpr int64_t kMostPositions = 1ll << 20;
// Pieces of a lookup: below, one per lane, from there on four. Rows of 1024 bf16 values, kernel time with one and with four: 256 rows 2.5 and 3.8 us,
// 2048 3.2 and 4.3, 4096 4.5 and 5.4, 8192 6.7 both (7.0 and 6.75 where nothing is cached); 65536 rows of 760 fp32 values 72.7 and 66.6.
constexpr int64_t kFewPieces = 1 << 20;

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
  ANC_REQUIRE(anc_apart(out, n * H * elem_size(out_type), table, V * H * elem_size(table_type)) && anc_apart(out, n * H * elem_size(out_type), ids, n * ids_bytes),
              "anc_embed_lookup: out overlaps an input");
  const int vec = table_type == ANC_F32 || out_type == ANC_F32 ? 4 : 8;
  const int64_t per_row = pieces_of(H, vec), most = kMostPieces / per_row;
  hipStream_t s = anc_stream(stream);
  AncProfScope prof(ANC_PROF_MISC, s);
  for (int64_t r = 0; r < n; r += most) {
    const int64_t rows = n - r < most ? n - r : most, total = rows * per_row;
    const int u = total >= kFewPieces ? 4 : 1;
    const bool once = n * H * elem_size(out_type) > kCached;
    const dim3 grid((unsigned)((total + u * kLookupLanes - 1) / (u * kLookupLanes)));
    with_type(table_type, [&](auto tt) {
      with_type(out_type, [&](auto to) {
        with_flag(H % vec != 0, [&](auto tail) {
          constexpr int TT = decltype(tt)::value, TO = decltype(to)::value;
          constexpr bool TAIL = decltype(tail)::value != 0;
          auto kernel = u == 1 ? k_embed_lookup<TT, TO, TAIL, 1, false>
                        : once ? k_embed_lookup<TT, TO, TAIL, 4, true> : k_embed_lookup<TT, TO, TAIL, 4, false>;
          hipLaunchKernelGGL(kernel, grid, dim3(kLookupLanes), 0, s, (const void *)(ids + (uint64_t)(r * ids_bytes)), ids_bytes == 8,
                             (uint32_t)total, V, fast_div((uint32_t)per_row), H, scale, (const elem_t<TT> *)table,
                             (elem_t<TO> *)out + r * H);
        });
      });
    });
  }
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
  for (int64_t edge : {kSub8Most, kSub16Most})
    if (edge < M && dw_chunks(edge) > most) most = dw_chunks(edge);
  return most * 2 * dw_pitch(H) * 4;
}

extern "C" int anc_embed_dw(uint64_t srt, uint64_t start, uint64_t cnt, uint64_t key, uint64_t grp, int64_t n, uint64_t dy, int dy_type,
                            int64_t H, float scale, uint64_t out, uint64_t compact, int64_t V, uint64_t workspace,
                            int64_t workspace_bytes, uint64_t stream) {
  ANC_REQUIRE(n >= 0 && n <= kMostPositions && H > 0 && H <= (1ll << 20) && V > 0 && V < (1ll << 31), "anc_embed_dw: n=%lld (at most %lld), V=%lld, H=%lld",
              (long long)n, (long long)kMostPositions, (long long)V, (long long)H);
  ANC_REQUIRE(type_ok(dy_type), "anc_embed_dw: type %d", dy_type);
  ANC_REQUIRE((out != 0) != (compact != 0), "anc_embed_dw: one of out and compact");
  if (n == 0) return ANC_OK;
  ANC_REQUIRE(srt && start && cnt && key && grp && dy && workspace, "anc_embed_dw: null pointer");
  ANC_REQUIRE(((srt | start | cnt | key | grp | out | compact) & 3) == 0 && dy % (uint64_t)elem_size(dy_type) == 0 && (workspace & 15) == 0,
              "anc_embed_dw: misaligned pointers");
  const int64_t chunks = dw_chunks(n), need = chunks * 2 * dw_pitch(H) * 4;
  ANC_REQUIRE(workspace_bytes >= need, "anc_embed_dw: workspace holds %lld bytes, %lld needed", (long long)workspace_bytes, (long long)need);
  const uint64_t to = out != 0 ? out : compact;       // (a compact gradient is n rows at most)
  const int64_t to_bytes = (out != 0 ? V : n) * H * 4, dy_bytes = n * H * elem_size(dy_type);
  ANC_REQUIRE(anc_outputs_apart({{to, to_bytes}, {workspace, need}, {dy, dy_bytes}, {srt, 4 * n}, {start, 4 * n}, {cnt, 4 * n}, {key, 4 * n}, {grp, 4 * n}}, 2),
              "anc_embed_dw: the gradient or the workspace overlaps another buffer");
  hipStream_t s = anc_stream(stream);
  AncProfScope prof(ANC_PROF_MISC, s);
  const EmbedDw p{(const int32_t *)srt, (const int32_t *)start, (const int32_t *)cnt, (const int32_t *)key, (const int32_t *)grp,
                  n, V, H, dw_pitch(H), dw_sub(n), dw_chunk(n), scale, (float *)out, (float *)compact, (float *)workspace};
  const bool once = n * H * elem_size(dy_type) > kCached;
  with_type(dy_type, [&](auto t) {
    with_flag(H % piece_of<decltype(t)::value, decltype(t)::value> != 0, [&](auto tail) {
      constexpr int T = decltype(t)::value, VEC = piece_of<T, T>;
      constexpr bool TAIL = decltype(tail)::value != 0;
      // (a team is at most 1024 columns wide: 32 KiB of LDS for the edges; one of few positions has one wavefront: 64 KiB)
      const bool few = n <= kFewMost;
      const int64_t waves = (H + 64 * VEC - 1) / (64 * VEC), widest = few ? 1 : 1024 / (64 * VEC), wide = waves < widest ? waves : widest;
      const int subs = few ? kFewSubs : kSubs;
      auto kernel = few ? (out != 0 ? k_embed_dw<T, TAIL, true, false, kFewSubs> : k_embed_dw<T, TAIL, false, false, kFewSubs>)
                    : out != 0 ? (once ? k_embed_dw<T, TAIL, true, true, kSubs> : k_embed_dw<T, TAIL, true, false, kSubs>)
                               : (once ? k_embed_dw<T, TAIL, false, true, kSubs> : k_embed_dw<T, TAIL, false, false, kSubs>);
      hipLaunchKernelGGL(kernel, dim3((unsigned)chunks, (unsigned)((waves + wide - 1) / wide)), dim3((unsigned)(64 * wide), subs),
                         (unsigned)(subs * 2 * 64 * wide * VEC * sizeof(float)), s, p, (const elem_t<T> *)dy);
    });
  });
  if (chunks > 1)
    with_flag(H % 4 != 0, [&](auto tail) {
      hipLaunchKernelGGL((k_embed_dw_join<decltype(tail)::value != 0>), dim3((unsigned)(chunks - 1), (unsigned)((H + 255) / 256)), dim3(kDwLanes), 0,
                         s, p);
    });
  ANC_LAUNCH_CHECK();
  return ANC_OK;
}
