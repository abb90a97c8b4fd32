// The gated feed-forward block between two residual additions, dense or over tokens sorted by expert (anc_route), as four products:
//
//   gated   h = silu(x Wg) * (x Wu)                     x (rows, H), Wg, Wu (H, I), h (rows, I); optionally the pre-activations g, u
//   down    y = h Wd + residual                         Wd (I, H)
//   grad    dh = dy Wd^T;  dg = dh u s (1 + g (1 - s)), du = dh g s, h = g s u, s = sigmoid(g)
//   dx      dx = dg Wg^T + du Wu^T + residual
//
// Weights lie (in, out), one after the other per expert, as the optimizer keeps its bf16 copies: forwards the contraction runs down their
// columns, whose fragments come from transposing LDS reads, backwards along their rows, so no transposed copy exists. Products of bf16
// accumulate in fp32 over ascending k (dx: all of dg, then all of du); each output is rounded once.
//
// k_ffn_tiles: a workgroup owns TM x TN values of the product (gated: half of the columns of either weight, so that a lane holds g and u of
// the same element) and runs k through LDS in stages of 64 or 32; wavefronts of 128 x 64, 64 x 128, 64 x 64 or 32 x 64. Operands go straight
// to LDS through descriptors that end with the segment or the matrix: rows and columns beyond read zeros and are not stored. What bounds
// its loop is the operands' way into LDS: a CU has some 64 lines under way at a time, so a line of 128 bytes asked for in halves, a step of 32 k
// apart, counts twice. Steps of 64 ask for whole lines of what lies along k (8192 rows, dx, 1024 x 2816, 128x128 tiles: 129 us in steps of 32,
// 100 in steps of 64; 2048 x 2048, 256x256: 130 and 120, 1.15 PFLOP/s; gated, 256x256: 131 and 116 to 125). Forwards 128x256 keeps steps of 32, of
// which two workgroups fit a CU and hide each other's ends (8192 rows, 1024 x 2816, gated: 107 us, one workgroup in steps of 64 143); backwards
// one of eight wavefronts in three stages of 64 beats them (64 experts of 1024 x 768, 16384 rows: dx 101 and 93). A CU takes in some 60 bytes a
// nanosecond so, which is why few tiles are small ones. What is left then is the outputs' bytes, which overlap little with the loops.
// k_ffn_few: 16 to 64 rows of a segment by 16 to 64 columns, the eight wavefronts of a workgroup taking every eighth step of k, each
// with stages of its own and no barrier, and adding up at the end in a fixed order: with few rows the weights' bytes are the work, and
// this way they are spread over as many CUs as there are.
#include "lds_dma.h"
#include "ns_common.h"

namespace {

template <int V> struct IC { static constexpr int value = V; };
enum { kGated, kDown, kGrad, kDx };
constexpr int TK = 32;

struct Ffn {
  const uint16_t *A[2], *B[2];          // (rows, K) and per expert (K, N) forwards, (N, K) backwards
  const int32_t *counts, *offsets;      // null: one segment of all rows
  int64_t rows;                         // dense: rows; else slots
  int K, N, experts, tn;                // tn: tiles side by side
  const void *residual;
  void *y;                              // down, dx; h otherwise
  const uint16_t *gate, *up;
  uint16_t *dgate, *dup;                // grad; gated: gate and up, null where not wanted
  int y_f32;
};

typedef float f32x4v __attribute__((ext_vector_type(4)));

// Where a workgroup's tile lies: the expert, its first row in the buffers and how many of the segment's rows are left from there.
struct Place { int e, n; int64_t row; int left; };

// Sums over lanes 0 .. lane of a wavefront.
__device__ __forceinline__ int sums_up_to(int v) {
  const int lane = (int)(threadIdx.x & 63);
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int o = __shfl_up(v, off, 64);
    v += lane >= off ? o : 0;
  }
  return v;
}

// Workgroup id -> tile. The tiles of all segments, TM rows each, are counted on the device, 64 experts at a time (the first 64 stay in registers);
// ids go round the XCDs in equal runs, a run in blocks of 8 row tiles by all columns, so that what an XCD works on at a time shares its L2.
__device__ __forceinline__ bool place_of(const Ffn &p, int TM, Place &at) {
  const int lane = (int)(threadIdx.x & 63);
  // (a segment stays inside its buffers, whatever the arrays hold)
  auto segment = [&](int e, int &first, int &count) {
    first = count = 0;
    if (e >= p.experts) return;
    const int64_t o = p.offsets[e], f = o < 0 ? 0 : o < p.rows ? o : p.rows, room = p.rows - f;
    const int n = p.counts[e];
    first = (int)f;
    count = n < 0 ? 0 : n < room ? n : (int)room;
  };
  int total, first = 0, count = 0, tiles = 0, upto = 0;
  if (p.counts == nullptr) {
    total = (int)((p.rows + TM - 1) / TM);
  } else {
    segment(lane, first, count);
    tiles = (count + TM - 1) / TM;
    upto = sums_up_to(tiles);
    total = __builtin_amdgcn_readlane(upto, 63);
    for (int c = 64; c < p.experts; c += 64) {
      int f, n;
      segment(c + lane, f, n);
      total += __builtin_amdgcn_readlane(sums_up_to((n + TM - 1) / TM), 63);
    }
  }
  const int all = total * p.tn, share = (all + kXcds - 1) / kXcds, b = (int)blockIdx.x, q = b / kXcds;
  const int id = b % kXcds * share + q;
  if (q >= share || id >= all) return false;
  const int group = id / (8 * p.tn), in = id - group * 8 * p.tn, high = total - group * 8 < 8 ? total - group * 8 : 8;
  const int m = group * 8 + in % high;
  at.n = in / high;
  if (p.counts == nullptr) {
    at.e = 0;
    at.row = (int64_t)m * TM;
    at.left = (int)(p.rows - at.row < 0x7FFFFFFF ? p.rows - at.row : 0x7FFFFFFF);
    return true;
  }
  int before = 0, c = 0;
  uint64_t hit;
  while ((hit = __ballot(upto > m - before && upto - tiles <= m - before)) == 0) {
    before += __builtin_amdgcn_readlane(upto, 63);
    c += 64;
    if (c >= p.experts) return false;
    segment(c + lane, first, count);
    tiles = (count + TM - 1) / TM;
    upto = sums_up_to(tiles);
  }
  const int l = __builtin_ctzll(hit), mine = m - before - __builtin_amdgcn_readlane(upto - tiles, l);
  at.e = c + l;
  at.row = (int64_t)__builtin_amdgcn_readlane(first, l) + (int64_t)mine * TM;
  at.left = __builtin_amdgcn_readlane(count, l) - mine * TM;
  return at.left > 0;
}

// One operand: where the next stage starts and how many bytes may be read from there on.
struct Feed {
  const char *at;
  int64_t left, step;
  __device__ __forceinline__ anc_i32x4 desc() const {
    return buffer_of(at, left <= 0 ? 0u : left < 0x7FFFFFF0ll ? (uint32_t)left : 0x7FFFFFF0u);
  }
  __device__ __forceinline__ void next() { at += step; left -= step; }
};
constexpr uint32_t kNowhere = 0x80000000u;                 // an offset beyond every descriptor

__device__ __forceinline__ float sigmoid(float g) { return __builtin_amdgcn_rcpf(1.0f + __expf(-g)); }
__device__ __forceinline__ void eight(const anc_u32x4 &q, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(q[i] << 16);
    f[2 * i + 1] = __uint_as_float(q[i] & 0xFFFF0000u);
  }
}
template <bool ONCE, typename V> __device__ __forceinline__ void put(V *p, const V &v) {
  if constexpr (ONCE) anc_st_stream(p, v);
  else *p = v;
}
template <bool ONCE> __device__ __forceinline__ void put_eight(uint16_t *p, const float (&f)[8]) {
  put<ONCE>((anc_u32x4 *)p, anc_u32x4{anc_pk_bf16(f[0], f[1]), anc_pk_bf16(f[2], f[3]), anc_pk_bf16(f[4], f[5]), anc_pk_bf16(f[6], f[7])});
}
// What eight values of the outputs take besides the product: gate and up, or the residual (fp32: both halves).
struct Side { anc_u32x4 a, b; };
template <int MODE> __device__ __forceinline__ Side side_of(const Ffn &p, int64_t at) {
  Side s{};
  if constexpr (MODE == kGrad) {
    s.a = *(const anc_u32x4 *)(p.gate + at);
    s.b = *(const anc_u32x4 *)(p.up + at);
  } else if constexpr (MODE != kGated) {
    if (p.residual != nullptr) {
      if (p.y_f32) {
        s.a = *(const anc_u32x4 *)((const float *)p.residual + at);
        s.b = *(const anc_u32x4 *)((const float *)p.residual + at + 4);
      } else {
        s.a = *(const anc_u32x4 *)((const uint16_t *)p.residual + at);
      }
    }
  }
  return s;
}
// Eight neighbouring values of the product (gated: of both) at element `at` of the outputs. ONCE: past the caches.
template <int MODE, bool ONCE> __device__ __forceinline__ void finish(const Ffn &p, int64_t at, float (&v)[8], const float (&w)[8], const Side &side) {
  if constexpr (MODE == kGated) {
    float h[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) h[k] = v[k] * sigmoid(v[k]) * w[k];
    put_eight<ONCE>((uint16_t *)p.y + at, h);
    if (p.dgate != nullptr) put_eight<ONCE>(p.dgate + at, v);
    if (p.dup != nullptr) put_eight<ONCE>(p.dup + at, w);
  } else if constexpr (MODE == kGrad) {
    float g[8], u[8], dg[8], du[8], h[8];
    eight(side.a, g);
    eight(side.b, u);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float s = sigmoid(g[k]), a = g[k] * s;
      dg[k] = v[k] * u[k] * (s * (1.0f + g[k] * (1.0f - s)));
      du[k] = v[k] * a;
      h[k] = a * u[k];
    }
    put_eight<ONCE>(p.dgate + at, dg);
    put_eight<ONCE>(p.dup + at, du);
    if (p.y != nullptr) put_eight<ONCE>((uint16_t *)p.y + at, h);
  } else if (p.y_f32) {
    anc_f32x4 a = {v[0], v[1], v[2], v[3]}, b = {v[4], v[5], v[6], v[7]};
    if (p.residual != nullptr) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        a[k] += __uint_as_float(side.a[k]);
        b[k] += __uint_as_float(side.b[k]);
      }
    }
    put<ONCE>((anc_f32x4 *)((float *)p.y + at), a);
    put<ONCE>((anc_f32x4 *)((float *)p.y + at + 4), b);
  } else {
    if (p.residual != nullptr) {
      float r[8];
      eight(side.a, r);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] += r[k];
    }
    put_eight<ONCE>((uint16_t *)p.y + at, v);
  }
}

// ---------------------------------------------------------------- many rows
// TM x TN values to a workgroup, WM x WN to a wavefront, WAVES wavefronts to a SIMD; fragments are read AHEAD slices of 16 k before their products:
// two where a wavefront has only two products to a slice, which do not cover a read (dx, 2048 rows of 1024 x 2816: 40.6 -> 37.2 us).
template <int MODE, int TM, int TN, int WM, int WN, int STEP, int STAGES, int WAVES, int AHEAD>
__global__ void __launch_bounds__(TM / WM * (TN / WN) * 64, WAVES) k_ffn_tiles(Ffn p) {
  constexpr bool kForward = MODE == kGated || MODE == kDown;
  constexpr int kWide = TN / WN, kWaves = TM / WM * kWide, kHigh = WM / 32, kAcross = WN / 32;       // wavefronts side by side, in all; fragments of A, of B
  constexpr int kRowA = STEP * 2, kBytesA = TM * kRowA, kBytesB = TN * kRowA, kStage = kBytesA + kBytesB, kStages = STAGES, kSlices = STEP / 16;
  constexpr int kPiecesA = kBytesA / 1024 / kWaves, kPiecesB = kBytesB / 1024 / kWaves, kPieces = kPiecesA + kPiecesB;
  constexpr int kCols = MODE == kGated ? TN / 2 : TN;       // columns of the outputs
  // Forwards the B tile is [STEP][kSub columns] once or twice: of either weight, or side by side.
  constexpr int kSub = MODE == kGated ? TN / 2 : 128, kRowB = kSub * 2, kRows = 1024 / kRowB, kSubPieces = STEP / kRows;
  static_assert((MODE == kGated || WN == 64) && kWaves * 8192 <= kStages * kStage && kPiecesA * kWaves * 1024 == kBytesA && kPiecesB * kWaves * 1024 == kBytesB,
                "room for the way out; whole pieces");
  __shared__ __attribute__((aligned(1024))) unsigned char ring[kStages * kStage];
  Place at;
  if (!place_of(p, TM, at)) return;
  const int K = p.K, N = p.N, lane = (int)(threadIdx.x & 63), wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int wm = wave / kWide, wn = wave % kWide, n0 = at.n * kCols;
  const int rows = at.left < TM ? at.left : TM, steps = (K + STEP - 1) / STEP, all = MODE == kDx ? 2 * steps : steps;

  const int half = wave * kPiecesB / kSubPieces;           // the part of the B tile that this wavefront fetches
  Feed fa, fb;
  auto term = [&](int t) {
    fa = Feed{(const char *)(p.A[t] + at.row * K), (int64_t)rows * K * 2, kRowA};
    if constexpr (kForward) {
      const int col = MODE == kGated ? n0 : n0 + half * kSub;
      fb = Feed{(const char *)(p.B[MODE == kGated ? half : 0] + (int64_t)at.e * K * N + col), ((int64_t)K * N - col) * 2, (int64_t)STEP * N * 2};
    } else {
      const int high = N - n0 < TN ? N - n0 : TN;
      fb = Feed{(const char *)(p.B[t] + ((int64_t)at.e * N + n0) * K), (int64_t)high * K * 2, kRowA};
    }
  };
  term(0);
  // Offsets of the pieces, 1 KiB of LDS each. Rows of 64 bytes: 16 to a piece, their four 16-byte chunks XORed with (row >> 2) & 3; of 128
  // 8, with row & 7. Forwards, B's rows of 256 bytes: 4 to a piece, with 4 * (row & 3); of 128: 8, with 4 * ((row >> 1) & 1). So the rows that a
  // read touches fall into different banks. Of a row's last step the chunks beyond K are sent nowhere, which reads zeros.
  constexpr int kLanes = kRowA / 16;                        // of a row
  const int chunk = STEP == 32 ? (lane & 3) ^ (lane >> 4) : (lane & 7) ^ (lane >> 3);
  const uint32_t beyond = chunk * 8 >= K - (steps - 1) * STEP ? kNowhere : 0u;
  uint32_t va[kPiecesA], vb[kPiecesB];
#pragma unroll
  for (int i = 0; i < kPiecesA; ++i) va[i] = (uint32_t)(((wave * kPiecesA + i) * (64 / kLanes) + lane / kLanes) * K * 2 + chunk * 16);
#pragma unroll
  for (int i = 0; i < kPiecesB; ++i) {
    const int piece = wave * kPiecesB + i;
    if constexpr (kForward) {
      const int row = lane / (kRowB / 16), key = kSub == 128 ? (row & 3) << 2 : (row >> 1 & 1) << 2;
      vb[i] = (uint32_t)((piece % kSubPieces * kRows + row) * N * 2 + ((lane % (kRowB / 16)) ^ key) * 16);
    } else {
      vb[i] = (uint32_t)((piece * (64 / kLanes) + lane / kLanes) * K * 2 + chunk * 16);
    }
  }
  int fetched = 0;
  uint32_t mask = steps == 1 ? beyond : 0u;
  auto issue = [&](int i, const anc_i32x4 &da, const anc_i32x4 &db, unsigned char *stage) {
    if (i < kPiecesA) dma16_bounded(da, va[i] | mask, lds_addr(stage + (wave * kPiecesA + i) * 1024));
    else dma16_bounded(db, kForward ? vb[i - kPiecesA] : vb[i - kPiecesA] | mask, lds_addr(stage + kBytesA + (wave * kPiecesB + i - kPiecesA) * 1024));
  };
  auto advance = [&]() {
    ++fetched;
    if (MODE == kDx && fetched == steps) term(1);
    else if (fetched >= all) fa.left = fb.left = 0;
    else { fa.next(); fb.next(); }
    const int k = MODE == kDx && fetched >= steps ? fetched - steps : fetched;
    mask = k == steps - 1 ? beyond : 0u;
  };

  // Columns of fragment j: gated, the first half are of Wg, the others the same ones of Wu, so that a lane holds g and u of one element.
  int ta, tb[kAcross];
  ta = (wm * WM + (lane & 31)) * kRowA;
  if constexpr (kForward) {
    const int s16 = lane & 15, g16 = lane >> 4, row = 8 * (g16 >> 1) + (s16 >> 2), key = kSub == 128 ? (row & 3) << 2 : (row >> 1 & 1) << 2;
#pragma unroll
    for (int j = 0; j < kAcross; ++j) {
      const int sub = MODE == kGated ? j / (kAcross / 2) : wn * WN / kSub;
      const int col = MODE == kGated ? wn * (WN / 16) + j % (kAcross / 2) * 4 : wn * WN % kSub / 8 + j * 4;     // (in chunks)
      tb[j] = kBytesA + sub * (STEP * kRowB) + row * kRowB + (((col + 2 * (g16 & 1) + ((s16 & 3) >> 1)) ^ key) * 16) + (s16 & 1) * 8;
    }
  } else {
#pragma unroll
    for (int j = 0; j < kAcross; ++j) tb[j] = kBytesA + (wn * WN + j * 32 + (lane & 31)) * kRowA;
  }
  f32x16 acc[kHigh][kAcross];
#pragma unroll
  for (int i = 0; i < kHigh; ++i)
#pragma unroll
    for (int j = 0; j < kAcross; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;

  constexpr int kLoads = kHigh + kAcross, kProducts = kHigh * kAcross;
  constexpr int kSets = AHEAD == 1 ? 2 : 4;
  bf16x8 a[kSets][kHigh], c[kSets][kAcross];
  // fragment i (b0 b1 .. a0 a1 ..) of k 16 kk .. 16 kk + 15 of a stage
  auto load = [&](int set, int i, const unsigned char *stage, int kk) {
    const int sw = ((kk * 2 + (lane >> 5)) ^ (STEP == 32 ? (lane >> 2) & 3 : lane & 7)) * 16;
    if (i >= kAcross) a[set][i - kAcross] = *(const bf16x8 *)(stage + ta + (i - kAcross) * (32 * kRowA) + sw);
    else if constexpr (kForward) c[set][i] = anc_lds_tr_frag(stage + tb[i] + kk * (16 * kRowB), stage + tb[i] + kk * (16 * kRowB) + 4 * kRowB);
    else c[set][i] = *(const bf16x8 *)(stage + tb[i] + sw);
  };
  auto multiply = [&](int set, int idx) {        // operands exchanged: a lane holds runs of 4 columns of one row
    f32x16 &to = acc[idx / kAcross][idx % kAcross];
    to = __builtin_amdgcn_mfma_f32_32x32x16_bf16(c[set][idx % kAcross], a[set][idx / kAcross], to, 0, 0, 0);
  };
  for (int i = 0; i < kStages; ++i) {
    const anc_i32x4 da = fa.desc(), db = fb.desc();
#pragma unroll
    for (int q = 0; q < kPieces; ++q) issue(q, da, db, ring + i * kStage);
    advance();
  }
  wait_vm<(kStages - 1) * kPieces>();
  lds_barrier();
#pragma unroll
  for (int kk = 0; kk < AHEAD; ++kk)
#pragma unroll
    for (int i = 0; i < kLoads; ++i) load(kk, i, ring, kk);
  // One step, a slice at a time: its products over the reads of a later one. Before the first reads of the next stage every wavefront has read this
  // one and the next has landed for all; the products from there on also go over the fetches into the place just read.
  // The last steps fetch nothing, the very last waits for nothing (1 to 5 % of a call, 3000 rows of 648 x 392 and 8 experts: dx 16.4 -> 15.7 us).
  auto step = [&](auto left, unsigned char *here, unsigned char *next) {
    constexpr int kLeft = decltype(left)::value;              // steps behind this one, kStages where there are as many or more
    constexpr bool kFetch = kLeft >= kStages, kMore = kLeft > 0;
    static_assert(kSlices % kSets == 0 && AHEAD < kSets, "a slice's fragments have one place");
    anc_i32x4 da, db;
#pragma unroll
    for (int kk = 0; kk < kSlices; ++kk) {
      if (kMore && kk == kSlices - AHEAD) {
        wait_vm<(kLeft < kStages - 1 ? kLeft - 1 : kStages - 2) * kPieces>();
        lds_barrier();
        if constexpr (kFetch) {
          da = fa.desc();
          db = fb.desc();
        }
      }
#pragma unroll
      for (int i = 0; i < kProducts; ++i) {
        multiply(kk % kSets, i);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int q = i; q < kLoads; q += kProducts) {
          if (kk + AHEAD < kSlices) load((kk + AHEAD) % kSets, q, here, kk + AHEAD);
          else if (kMore) load((kk + AHEAD) % kSets, q, next, kk + AHEAD - kSlices);
        }
        if (kFetch && kk >= kSlices - AHEAD) {
#pragma unroll
          for (int q = (kk - (kSlices - AHEAD)) * kProducts + i; q < kPieces; q += AHEAD * kProducts) issue(q, da, db, here);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if constexpr (kFetch) advance();
  };
  int here = 0;
  auto forth = [&](auto left) {
    const int next = here + kStage < kStages * kStage ? here + kStage : 0;
    step(left, ring + here, ring + next);
    here = next;
  };
  for (int t = kStages; t < all; ++t) forth(IC<kStages>{});
  if constexpr (kStages > 2)
    if (all > 2) forth(IC<2>{});
  if (all > 1) forth(IC<1>{});
  forth(IC<0>{});
  wait_vm<0>();                                  // (zeros that a short k left on their way into the stages)
  lds_barrier();

  unsigned char *r = ring + wave * 8192;
  const int rr = lane & 31, hh = lane >> 5;
  if constexpr (MODE == kGated) {
    // A lane holds g and u of the same elements: h, g and u leave it as bf16, 32 rows at a time through LDS, so that a wavefront of 64 columns stores
    // whole lines of 128 bytes, past the caches, which keep the operands of the tiles still to come. (Half lines past the caches: 3.6 TB/s, whole ones
    // 5.4; through them 5.7 both. 32 columns to a wavefront go through them.)
    constexpr int kReal = WN / 2, kChunks = kReal / 8, kLine = kReal * 2;
    auto out = [&](int i, uint16_t *to, auto value) {
#pragma unroll
      for (int j = 0; j < kAcross / 2; ++j)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          float v[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] = value(acc[i][j][4 * g + k], acc[i][j + kAcross / 2][4 * g + k]);
          *(anc_u32x2 *)(r + rr * kLine + (((j * 4 + g) ^ (rr & (kChunks - 1))) * 16) + hh * 8) = anc_u32x2{anc_pk_bf16(v[0], v[1]), anc_pk_bf16(v[2], v[3])};
        }
      lds_wave_sync();
#pragma unroll
      for (int z = 0; z < kChunks / 2; ++z) {
        const int idx = z * 64 + lane, row = idx / kChunks, ch = idx % kChunks, in = wm * WM + i * 32 + row, col = n0 + wn * kReal + ch * 8;
        const anc_u32x4 v = *(const anc_u32x4 *)(r + row * kLine + ((ch ^ (row & (kChunks - 1))) * 16));
        if (in < rows && col < N) put<kLine == 128>((anc_u32x4 *)(to + (at.row + in) * N + col), v);
      }
      lds_wave_sync();
    };
#pragma unroll
    for (int i = 0; i < kHigh; ++i) {
      out(i, (uint16_t *)p.y, [](float g, float u) { return g * sigmoid(g) * u; });
      if (p.dgate != nullptr) out(i, p.dgate, [](float g, float) { return g; });
      if (p.dup != nullptr) out(i, p.dup, [](float, float u) { return u; });
    }
  } else {
    // Out through LDS, 32 rows of 64 values at a time: a lane then holds 8 neighbouring columns of a row. What the outputs take besides the
    // product is fetched one such block ahead; results leave past the caches.
    const int col0 = n0 + wn * 64;
    Side side[2][4];
    auto where = [&](int i, int z, int64_t &e) {
      const int idx = z * 64 + lane, in = wm * WM + i * 32 + idx / 8, col = col0 + idx % 8 * 8;
      e = (at.row + in) * N + col;
      return in < rows && col < N;
    };
    auto fetch = [&](int i) {
#pragma unroll
      for (int z = 0; z < 4; ++z) {
        int64_t e;
        if (where(i, z, e)) side[i & 1][z] = side_of<MODE>(p, e);
      }
    };
    fetch(0);
#pragma unroll
    for (int i = 0; i < kHigh; ++i) {
#pragma unroll
      for (int j = 0; j < kAcross; ++j)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *(anc_f32x4 *)(r + rr * 256 + (((j * 8 + 2 * g + hh) ^ (rr & 15)) * 16)) =
              anc_f32x4{acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
      lds_wave_sync();
      if (i + 1 < kHigh) fetch(i + 1);
#pragma unroll
      for (int z = 0; z < 4; ++z) {
        const int idx = z * 64 + lane, row = idx / 8, ch = idx % 8 * 2;
        const anc_f32x4 lo = *(const anc_f32x4 *)(r + row * 256 + ((ch ^ (row & 15)) * 16)), hi = *(const anc_f32x4 *)(r + row * 256 + (((ch + 1) ^ (row & 15)) * 16));
        float v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
        int64_t e;
        if (where(i, z, e)) finish<MODE, true>(p, e, v, v, side[i & 1][z]);
      }
      lds_wave_sync();
    }
  }
}

// ---------------------------------------------------------------- few rows
// R blocks of 16 rows by C blocks of 16 columns (gated: half of them of either weight), as many stages as LDS holds: what bounds a short
// product is how many of its weights' bytes are under way at a time.
template <int MODE, int R, int C> __global__ void __launch_bounds__(512, 2) k_ffn_few(Ffn p) {
  constexpr bool kForward = MODE == kGated || MODE == kDown;
  constexpr int TM = 16 * R, kWaves = 8, kPieces = R + C, kStage = kPieces * 1024, kStages = 18 / kPieces;
  constexpr int kSub = MODE == kGated ? C / 2 : C;          // blocks of a row of one weight
  constexpr int kRowB = kSub * 32, kPer = 1024 / kRowB;     // bytes of it, rows to a piece
  constexpr int kCols = kSub * 16;
  __shared__ __attribute__((aligned(1024))) unsigned char ring[kWaves * kStages * kStage];
  static_assert(kWaves * R * C * 1024 <= (int)sizeof(ring) && kStages >= 2 && sizeof(ring) <= 147456, "room for the partial sums");
  Place at;
  if (!place_of(p, TM, at)) return;
  const int K = p.K, N = p.N, lane = (int)(threadIdx.x & 63), wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int n0 = at.n * kCols, rows = at.left < TM ? at.left : TM, steps = (K + TK - 1) / TK, all = MODE == kDx ? 2 * steps : steps;
  unsigned char *mine = ring + wave * kStages * kStage;
  const int chunk = (lane & 3) ^ (lane >> 4);
  const uint32_t beyond = chunk * 8 >= K - (steps - 1) * TK ? kNowhere : 0u;
  const uint32_t va = (uint32_t)((lane >> 2) * K * 2 + chunk * 16);
  const uint32_t vb = kForward ? (uint32_t)(lane / (kRowB / 16) * N * 2 + lane % (kRowB / 16) * 16) : va;
  auto fetch = [&](int t, unsigned char *stage) {           // step t of all; beyond them nothing is read
    const int second = MODE == kDx && t >= steps, k = t - (second ? steps : 0), k0 = k * TK;
    const bool there = t < all;
    const uint32_t mask = k == steps - 1 ? beyond : 0u;
    const int64_t lefta = ((int64_t)rows * K - k0) * 2;
    const anc_i32x4 da = buffer_of((const char *)(p.A[second] + at.row * K + (there ? k0 : 0)), there ? (uint32_t)lefta : 0u);
#pragma unroll
    for (int i = 0; i < R; ++i) dma16_bounded(da, (va + (uint32_t)(i * 16 * K * 2)) | mask, lds_addr(stage + i * 1024));
    if constexpr (kForward) {
#pragma unroll
      for (int i = 0; i < C; ++i) {
        const int w = MODE == kGated ? i / (C / 2 > 0 ? C / 2 : 1) : 0, piece = MODE == kGated ? i % (C / 2 > 0 ? C / 2 : 1) : i;
        const Feed f{(const char *)(p.B[w] + (int64_t)at.e * K * N + (there ? (int64_t)k0 * N : 0) + n0), there ? ((int64_t)(K - k0) * N - n0) * 2 : 0, 0};
        dma16_bounded(f.desc(), vb + (uint32_t)(piece * kPer * N * 2), lds_addr(stage + (R + i) * 1024));
      }
    } else {
      const int high = N - n0 < kCols ? N - n0 : kCols;
      const anc_i32x4 db = buffer_of((const char *)(p.B[second] + ((int64_t)at.e * N + n0) * K + (there ? k0 : 0)), there ? (uint32_t)(((int64_t)high * K - k0) * 2) : 0u);
#pragma unroll
      for (int i = 0; i < C; ++i) dma16_bounded(db, (vb + (uint32_t)(i * 16 * K * 2)) | mask, lds_addr(stage + (R + i) * 1024));
    }
  };
  // A lane's eight values of the outputs.
  constexpr int kOcts = kCols / 8;
  static_assert(TM * kOcts <= kWaves * 64, "one each");
  const int row = (int)threadIdx.x / kOcts, oct = (int)threadIdx.x % kOcts, col = n0 + oct * 8;
  const bool ours = row < rows && col < N;
  const int64_t e = (at.row + row) * N + col;
  f32x4v acc[R][C];
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < C; ++j) acc[i][j] = f32x4v{0.0f, 0.0f, 0.0f, 0.0f};
  const int s16 = lane & 15, g16 = lane >> 4;
  const int ta = s16 * 64 + ((g16 ^ ((s16 >> 2) & 3)) * 16);
#pragma unroll 1
  for (int i = 0; i < kStages; ++i) fetch(wave + i * kWaves, mine + i * kStage);
  int here = 0;
  for (int t = wave; t < all; t += kWaves) {
    const unsigned char *stage = mine + here;
    // (behind the last step nothing is fetched, and the last stages wait for one another: 1 to 64 rows 0.4 us less than fetching zeros)
    if (t + (kStages - 1) * kWaves < all) wait_vm<(kStages - 1) * kPieces>();
    else wait_vm<0>();
    bf16x8 a[R], b[C];
#pragma unroll
    for (int i = 0; i < R; ++i) a[i] = *(const bf16x8 *)(stage + i * 1024 + ta);
#pragma unroll
    for (int j = 0; j < C; ++j) {
      if constexpr (kForward) {
        const unsigned char *q = stage + R * 1024 + j / kSub * (kSub * 1024) + (8 * g16 + (s16 >> 2)) * kRowB + j % kSub * 32 + (s16 & 3) * 8;
        b[j] = anc_lds_tr_frag(q, q + 4 * kRowB);
      } else {
        b[j] = *(const bf16x8 *)(stage + (R + j) * 1024 + ta);
      }
    }
    lds_wave_sync();                             // (read before the stage is fetched into again)
    if (t + kStages * kWaves < all) fetch(t + kStages * kWaves, mine + here);
#pragma unroll
    for (int j = 0; j < C; ++j)
#pragma unroll
      for (int i = 0; i < R; ++i) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[j], a[i], acc[i][j], 0, 0, 0);
    here = here + kStage < kStages * kStage ? here + kStage : 0;
  }
  const Side side = ours ? side_of<MODE>(p, e) : Side{};     // (on its way over the sums)
  wait_vm<0>();
  lds_barrier();
  // The wavefronts' sums, in ascending order: [wavefront][row][column] fp32. Where eight values to a lane leave lanes idle, all add up over the first
  // one's first (1 to 32 rows, 1024 -> 2816: gated 0.5 us less; 1024 rows, 64x64, where none are: down 0.6 more, so not there).
  float *sums = (float *)ring;
  constexpr int kSums = TM * C * 16, kParts = TM * kOcts < kWaves * 64 ? 1 : kWaves;
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < C; ++j) *(f32x4v *)(sums + wave * kSums + (i * 16 + s16) * (C * 16) + j * 16 + g16 * 4) = acc[i][j];
  lds_barrier();
  if constexpr (kParts == 1) {
    for (int idx = (int)threadIdx.x * 4; idx < rows * (C * 16); idx += kWaves * 256) {
      f32x4v v = *(const f32x4v *)(sums + idx);
#pragma unroll
      for (int w = 1; w < kWaves; ++w) v += *(const f32x4v *)(sums + w * kSums + idx);
      *(f32x4v *)(sums + idx) = v;
    }
    lds_barrier();
  }
  if (!ours) return;
  auto total = [&](int first, float (&f)[8]) {
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = sums[row * (C * 16) + first + k];
#pragma unroll
    for (int w = 1; w < kParts; ++w)
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] += sums[w * kSums + row * (C * 16) + first + k];
  };
  float v[8], w[8];
  total(oct * 8, v);
  if constexpr (MODE == kGated) total(kCols + oct * 8, w);
  finish<MODE, false>(p, e, v, w, side);
}

// ---------------------------------------------------------------- launch
// Which kernel takes a call: the one whose rounds take least by what a step of 32 k and a round cost, in us: of k_ffn_tiles where up to 128, 256,
// .. workgroups are at work; of k_ffn_few, one workgroup to a CU, for a wavefront's step (of eight). `most`: rows that all segments hold together at
// most. Fitted to whole calls (1 to 8192 rows, up to 2272 x 4096, dense; 3 to 128 experts of up to 1128 x 2128): over 35 calls of each kind the choice was
// 0.5 to 1.5 % off the best of the eight on average, before the backward pass's 128x256 tiles took their present form (its line was fitted again by
// itself). The tiles' side knows no weights' bytes: for larger experts with few rows each its ranking is a guess. Both sides of some lines, us:
//   gated, 1024 -> 2816: 64 rows: 32x32 by eight wavefronts 10.1, 128x128 tiles 13.8; 256 rows: 64x64 by eight wavefronts 23.4, 64x128 tiles 10.3, 128x128
//   15.0; 1024 rows: 128x128 22.7, 128x256 20.9; 2048 x 2048, 8192 rows: 128x256 125, 256x256 116
//   down, 2816 -> 1024: 1024 rows: 64x64 by eight wavefronts 17.8, 64x128 19.8, 128x128 32.7; 2048 rows 32.4, 20.1, 32.9; 8192 rows: 64x128 64, 128x128
//   49, 128x256 52, 256x256 68
//   grad, 512 rows of 1024 x 2816: 64x128 11.2, 128x128 17.0; dx, 2048 x 2048, 8192 rows, whole rounds: 256x256 121, 128x128 142; 1024 x 2816, half a round
//   of 256x256: 141, 128x128 100 or 114 by the buffers' places (no reason found), 128x256 92 to 102
//   grad of a short k, 57 experts of 104 x 2032, 87 rows each, where the outputs' bytes are the work: 64x128 35, 128x256 43
//   64 experts of 1024 x 768, 4 rows each, gated: 64x64 74, 128x128 40; 128 rows each, down: 128x256 37, 256x256, which just miss one round, 50
template <int MODE> int launch(Ffn p, int64_t most, const char *who, hipStream_t s) {
  constexpr bool kBack = MODE == kGrad || MODE == kDx;
  constexpr int per = MODE == kGated ? 2 : 1;                 // values of the product to one of the outputs
  const int64_t some = p.counts == nullptr ? 1 : most < p.experts ? most : p.experts;              // segments that can hold a row
  const float steps = (float)((p.K + TK - 1) / TK * (MODE == kDx ? 2 : 1));
  auto columns = [&](int64_t TN) { return (p.N + TN / per - 1) / (TN / per); };
  // workgroups that find work, about (an even routing leaves E e^(-most / E) experts without a row, an uneven one some above their share); and at most
  const int64_t used = p.counts == nullptr ? 1 : (int64_t)ceilf((float)p.experts * -expm1f(-(float)most / (float)p.experts));
  auto live = [&](int64_t TM, int64_t TN) {
    const int64_t m = p.counts == nullptr ? (most + TM - 1) / TM : most / TM + (used * 3 + 4) / 5;
    return (m < used ? used : m) * columns(TN);
  };
  auto grid_of = [&](int64_t TM) {
    const int64_t m = p.counts == nullptr ? (most + TM - 1) / TM : most / TM + some;
    return (m * p.tn + kXcds - 1) / kXcds * kXcds;
  };
  auto rounds = [&](int64_t n, int64_t slots, auto cost) { return (float)(n / slots) * cost(slots) + (n % slots ? cost(n % slots) : 0.0f); };
  const float cold = p.counts == nullptr ? 1.0f : 1.4f;      // every expert's weights come from memory, in short rows
  // The backward epilogue's ten bytes an element at 5.5 TB/s, and how much of them the other workgroups' loops leave uncovered.
  auto outputs = [&](int64_t r, int tile, float share) { return MODE == kGrad ? (float)r * (float)tile * 10.0f / 5.5e6f * share : 0.0f; };
  const float time[] = {
      rounds(live(256, 256), 256, [&](int64_t r) { return steps * (r <= 128 ? 0.75f : 0.92f) + (MODE == kGated ? 7.0f : 5.0f) + outputs(r, 256 * 256, 0.7f); }),
      kBack ? rounds(live(128, 256), 256, [&](int64_t r) { return steps * (r <= 128 ? 0.37f : 0.52f) + 4.0f + outputs(r, 128 * 256, 0.5f); })
            : rounds(live(128, 256), 512, [&](int64_t r) { return steps * (r <= 128 ? 0.46f : r <= 256 ? 0.60f : 0.98f) + 4.0f; }),
      MODE == kGated ? rounds(live(128, 128), 768, [&](int64_t r) { return steps * (r <= 128 ? 0.33f : r <= 256 ? 0.38f : r <= 512 ? 0.63f : 0.90f) + 3.5f; })
                     : rounds(live(128, 128), 512, [&](int64_t r) { return steps * (r <= 128 ? 0.33f : r <= 256 ? 0.37f : 0.57f) + 4.5f + outputs(r, 128 * 128, 0.4f); }),
      rounds(live(64, 128), 512, [&](int64_t r) { return steps * (r <= 256 ? 0.19f : 0.35f) + 4.5f + outputs(r, 64 * 128, 0.2f); }),
      rounds(live(64, 64), 256, [&](int64_t) { return cold * (steps / 8 * 0.90f + 7.7f); }),
      rounds(live(32, 64), 256, [&](int64_t) { return cold * (steps / 8 * 0.72f + 4.6f); }),
      rounds(live(32, 32), 256, [&](int64_t) { return cold * (steps / 8 * 0.47f + 4.2f); }),
      MODE == kGated ? 1e30f : rounds(live(16, 16), 256, [&](int64_t) { return cold * (steps / 8 * 0.25f + 4.0f); }),
  };
  int best = 0;
  for (int i = 1; i < 8; ++i)
    if (time[i] < time[best]) best = i;
  AncProfScope prof(ANC_PROF_MISC, s);
  auto few = [&](auto R, auto C) {
    constexpr int r = decltype(R)::value, c = decltype(C)::value;
    p.tn = (int)columns(16 * c);
    ANC_REQUIRE(grid_of(16 * r) < (1ll << 31) / 512, "%s: too large for one call", who);
    hipLaunchKernelGGL((k_ffn_few<MODE, r, c>), dim3((unsigned)grid_of(16 * r)), dim3(512), 0, s, p);
    return ANC_OK;
  };
  auto tiles = [&](auto TM, auto TN, auto WM, auto WN, auto ST, auto SG, auto W, auto AH) {
    constexpr int tm = decltype(TM)::value, tn = decltype(TN)::value, wm = decltype(WM)::value, wn = decltype(WN)::value, st = decltype(ST)::value, sg = decltype(SG)::value, w = decltype(W)::value, ah = decltype(AH)::value;
    p.tn = (int)columns(tn);
    ANC_REQUIRE(grid_of(tm) < (1ll << 31) / 512, "%s: too large for one call", who);
    hipLaunchKernelGGL((k_ffn_tiles<MODE, tm, tn, wm, wn, st, sg, w, ah>), dim3((unsigned)grid_of(tm)), dim3(tm / wm * (tn / wn) * 64), 0, s, p);
    return ANC_OK;
  };
  constexpr int kTall = MODE == kGated ? 64 : 128;            // a wavefront's rows; gated: 64 columns of either weight
  int rc = ANC_OK;
  switch (best) {
    case 0: rc = tiles(IC<256>{}, IC<256>{}, IC<kTall>{}, IC<8192 / kTall>{}, IC<64>{}, IC<2>{}, IC<2>{}, IC<1>{}); break;
    case 1:
      if constexpr (kBack) rc = tiles(IC<128>{}, IC<256>{}, IC<64>{}, IC<64>{}, IC<64>{}, IC<3>{}, IC<2>{}, IC<1>{});
      else rc = tiles(IC<128>{}, IC<256>{}, IC<kTall>{}, IC<8192 / kTall>{}, IC<32>{}, IC<3>{}, IC<2>{}, IC<1>{});
      break;
    case 2:
      if constexpr (MODE == kGated) rc = tiles(IC<128>{}, IC<128>{}, IC<64>{}, IC<64>{}, IC<32>{}, IC<3>{}, IC<3>{}, IC<1>{});
      else rc = tiles(IC<128>{}, IC<128>{}, IC<64>{}, IC<64>{}, IC<64>{}, IC<2>{}, IC<2>{}, IC<1>{});
      break;
    case 3: rc = tiles(IC<64>{}, IC<128>{}, IC<32>{}, IC<64>{}, IC<64>{}, IC<3>{}, IC<2>{}, IC<2>{}); break;
    case 4: rc = few(IC<4>{}, IC<4>{}); break;
    case 5: rc = few(IC<2>{}, IC<4>{}); break;
    case 6: rc = few(IC<2>{}, IC<2>{}); break;
    default: if constexpr (per == 1) rc = few(IC<1>{}, IC<1>{}); break;
  }
  if (rc != ANC_OK) return rc;
  ANC_LAUNCH_CHECK();
  return ANC_OK;
}

int check(const char *who, uint64_t counts, uint64_t offsets, int64_t experts, int64_t rows, int64_t tokens, int64_t H, int64_t I) {
  ANC_REQUIRE(H > 0 && I > 0 && H % 8 == 0 && I % 8 == 0 && H <= (1 << 17) && I <= (1 << 17),
              "%s: needs H %% 8 == 0 and I %% 8 == 0 (H=%lld I=%lld)", who, (long long)H, (long long)I);
  ANC_REQUIRE(rows >= 0 && rows < (1ll << 31), "%s: %lld rows", who, (long long)rows);
  ANC_REQUIRE((counts != 0) == (experts > 0) && (offsets != 0) == (experts > 0) && ((counts | offsets) & 3) == 0 && experts >= 0 && experts <= 512,
              "%s: bad segments (%lld experts)", who, (long long)experts);
  ANC_REQUIRE(tokens >= 0 && tokens <= rows && (experts > 0 || tokens == rows), "%s: %lld of %lld rows in segments", who, (long long)tokens, (long long)rows);
  return ANC_OK;
}
// Outputs meet no other buffer of the call, but for the pairs that are one buffer on purpose (the same elements, read before they are written).
template <int O, int I> int apart(const char *who, const AncSpan (&out)[O], const AncSpan (&in)[I], const int (&pair)[O]) {
  ANC_REQUIRE(anc_outputs_apart(out, O), "%s: outputs overlap", who);
  for (int i = 0; i < O; ++i)
    for (int j = 0; j < I; ++j)
      ANC_REQUIRE((pair[i] == j && out[i].at == in[j].at && out[i].bytes == in[j].bytes) || anc_apart(out[i].at, out[i].bytes, in[j].at, in[j].bytes),
                  "%s: an output overlaps an input", who);
  return ANC_OK;
}
AncSpan span(uint64_t at, int64_t bytes) { return AncSpan{at, at != 0 ? bytes : 0}; }

}  // namespace

extern "C" int anc_gated_ffn(uint64_t x, uint64_t Wg, uint64_t Wu, uint64_t counts, uint64_t offsets, int64_t experts, int64_t rows, int64_t tokens,
                             int64_t H, int64_t I, uint64_t h, uint64_t gate, uint64_t up, uint64_t stream) {
  const char *who = "anc_gated_ffn";
  if (int rc = check(who, counts, offsets, experts, rows, tokens, H, I)) return rc;
  if (tokens == 0) return ANC_OK;
  ANC_REQUIRE(x && Wg && Wu && h && ((x | Wg | Wu | h | gate | up) & 15) == 0, "%s: null or misaligned pointer", who);
  const int64_t E = experts > 0 ? experts : 1, w = E * H * I * 2, n = rows * I * 2;
  if (int rc = apart<3, 5>(who, {span(h, n), span(gate, n), span(up, n)},
                           {span(x, rows * H * 2), span(Wg, w), span(Wu, w), span(counts, 4 * experts), span(offsets, 4 * experts + 4)}, {-1, -1, -1})) return rc;
  Ffn p{};
  p.A[0] = (const uint16_t *)x;
  p.B[0] = (const uint16_t *)Wg;
  p.B[1] = (const uint16_t *)Wu;
  p.counts = (const int32_t *)counts;
  p.offsets = (const int32_t *)offsets;
  p.rows = rows;
  p.K = (int)H;
  p.N = (int)I;
  p.experts = (int)experts;
  p.y = (void *)h;
  p.dgate = (uint16_t *)gate;
  p.dup = (uint16_t *)up;
  return launch<kGated>(p, tokens, who, anc_stream(stream));
}

extern "C" int anc_ffn_down(uint64_t h, uint64_t Wd, uint64_t counts, uint64_t offsets, int64_t experts, int64_t rows, int64_t tokens, int64_t I,
                            int64_t H, uint64_t residual, uint64_t y, int y_type, uint64_t stream) {
  const char *who = "anc_ffn_down";
  if (int rc = check(who, counts, offsets, experts, rows, tokens, H, I)) return rc;
  ANC_REQUIRE(y_type == ANC_F32 || y_type == ANC_BF16, "%s: bad y_type %d", who, y_type);
  if (tokens == 0) return ANC_OK;
  ANC_REQUIRE(h && Wd && y && ((h | Wd | y | residual) & 15) == 0, "%s: null or misaligned pointer", who);
  const int64_t E = experts > 0 ? experts : 1, n = rows * H * (y_type == ANC_F32 ? 4 : 2);
  if (int rc = apart<1, 5>(who, {span(y, n)}, {span(residual, n), span(h, rows * I * 2), span(Wd, E * H * I * 2), span(counts, 4 * experts), span(offsets, 4 * experts + 4)}, {0})) return rc;
  Ffn p{};
  p.A[0] = (const uint16_t *)h;
  p.B[0] = (const uint16_t *)Wd;
  p.counts = (const int32_t *)counts;
  p.offsets = (const int32_t *)offsets;
  p.rows = rows;
  p.K = (int)I;
  p.N = (int)H;
  p.experts = (int)experts;
  p.residual = (const void *)residual;
  p.y = (void *)y;
  p.y_f32 = y_type == ANC_F32;
  return launch<kDown>(p, tokens, who, anc_stream(stream));
}

extern "C" int anc_gated_ffn_grad(uint64_t dy, uint64_t Wd, uint64_t gate, uint64_t up, uint64_t counts, uint64_t offsets, int64_t experts,
                                  int64_t rows, int64_t tokens, int64_t H, int64_t I, uint64_t dgate, uint64_t dup, uint64_t h, uint64_t stream) {
  const char *who = "anc_gated_ffn_grad";
  if (int rc = check(who, counts, offsets, experts, rows, tokens, H, I)) return rc;
  if (tokens == 0) return ANC_OK;
  ANC_REQUIRE(dy && Wd && gate && up && dgate && dup && ((dy | Wd | gate | up | dgate | dup | h) & 15) == 0, "%s: null or misaligned pointer", who);
  const int64_t E = experts > 0 ? experts : 1, n = rows * I * 2;
  if (int rc = apart<3, 6>(who, {span(dgate, n), span(dup, n), span(h, n)},
                           {span(gate, n), span(up, n), span(dy, rows * H * 2), span(Wd, E * H * I * 2), span(counts, 4 * experts), span(offsets, 4 * experts + 4)}, {0, 1, -1})) return rc;
  Ffn p{};
  p.A[0] = (const uint16_t *)dy;
  p.B[0] = (const uint16_t *)Wd;
  p.counts = (const int32_t *)counts;
  p.offsets = (const int32_t *)offsets;
  p.rows = rows;
  p.K = (int)H;
  p.N = (int)I;
  p.experts = (int)experts;
  p.gate = (const uint16_t *)gate;
  p.up = (const uint16_t *)up;
  p.dgate = (uint16_t *)dgate;
  p.dup = (uint16_t *)dup;
  p.y = (void *)h;
  return launch<kGrad>(p, tokens, who, anc_stream(stream));
}

extern "C" int anc_gated_ffn_dx(uint64_t dgate, uint64_t dup, uint64_t Wg, uint64_t Wu, uint64_t counts, uint64_t offsets, int64_t experts,
                                int64_t rows, int64_t tokens, int64_t H, int64_t I, uint64_t residual, uint64_t dx, int dx_type, uint64_t stream) {
  const char *who = "anc_gated_ffn_dx";
  if (int rc = check(who, counts, offsets, experts, rows, tokens, H, I)) return rc;
  ANC_REQUIRE(dx_type == ANC_F32 || dx_type == ANC_BF16, "%s: bad dx_type %d", who, dx_type);
  if (tokens == 0) return ANC_OK;
  ANC_REQUIRE(dgate && dup && Wg && Wu && dx && ((dgate | dup | Wg | Wu | dx | residual) & 15) == 0, "%s: null or misaligned pointer", who);
  const int64_t E = experts > 0 ? experts : 1, w = E * H * I * 2, n = rows * H * (dx_type == ANC_F32 ? 4 : 2);
  if (int rc = apart<1, 7>(who, {span(dx, n)}, {span(residual, n), span(dgate, rows * I * 2), span(dup, rows * I * 2), span(Wg, w), span(Wu, w), span(counts, 4 * experts), span(offsets, 4 * experts + 4)}, {0})) return rc;
  Ffn p{};
  p.A[0] = (const uint16_t *)dgate;
  p.A[1] = (const uint16_t *)dup;
  p.B[0] = (const uint16_t *)Wg;
  p.B[1] = (const uint16_t *)Wu;
  p.counts = (const int32_t *)counts;
  p.offsets = (const int32_t *)offsets;
  p.rows = rows;
  p.K = (int)I;
  p.N = (int)H;
  p.experts = (int)experts;
  p.residual = (const void *)residual;
  p.y = (void *)dx;
  p.y_f32 = dx_type == ANC_F32;
  return launch<kDx>(p, tokens, who, anc_stream(stream));
}
