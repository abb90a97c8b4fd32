// The experts' weight gradients over tokens sorted by expert (anc_route): for every expert e
//     dW[e] (K, N) (+)= sum over its tokens s of x[s]^T dy[s],   x (slots, K), dy (slots, N) bf16, fp32 accumulation.
// Segments are ragged and known on the device only, so the grid covers every expert's whole weight and a workgroup reads its segment.
//
// One workgroup owns 256x256 (or 128x256) outputs of one expert and runs the expert's tokens in ascending order, 32 a step, one
// accumulator per element: no split of the tokens, an expert's bits are a function of its own rows. Both operands lie token by token, and
// the product contracts over tokens, so tiles [32 tokens][columns] go straight to LDS, three stages of them, and the fragments
// come from transposing LDS reads. Rows past the segment's end and stages past the last are never fetched: the buffer descriptor of a
// stage ends with the segment, and loads beyond it give zeros. (Columns past K or N are the next row's: they meet outputs that are
// not stored.)
//
// What bounds it is the operands' way into LDS, some 13 bytes per clock and CU, then the outputs' bytes. One layer of 16 experts, three
// weights of 1024x1024 with bf16 copies, 16384 rows in segments of 1:4: 177 us with 128x256 tiles and the experts in their order, 8 tiles
// at a time to an XCD; 151 with the experts by falling length and 16 .. 32 tiles at a time, 138 with 256x256 tiles, 103 of them
// without the stores.
#include "lds_dma.h"
#include "ns_common.h"

namespace {

constexpr int TN = 256, TK = 32, kStages = 3, kRowB = TN * 2, kBytesB = TK * kRowB;
constexpr int kMostProblems = 8;

struct DwOne {
  const uint16_t *x, *dy;
  float *dW;
  uint16_t *g16;
  int K, N, tn, tiles;                                         // tiles of one expert, tn of them side by side
  int accumulate;
};
struct DwMulti {
  const int32_t *counts, *offsets, *order;
  int64_t capacity;                                            // slots
  int count, experts, unit;                                    // tiles that follow each other on one XCD
  int unit0[kMostProblems + 1];                                // first unit of each problem among an expert's
  DwOne p[kMostProblems];
};

// One operand's rows of a tile: where the next stage starts and how many bytes of the segment are left from there.
struct Feed {
  const char *at;
  int64_t left, step;
  __device__ __forceinline__ anc_i32x4 desc() const {
    return buffer_of(at, left <= 0 ? 0u : left < 0xFFFFFFFFll ? (uint32_t)left : 0xFFFFFFFFu);
  }
  __device__ __forceinline__ void next() { at += step; left -= step; }
};

// Wavefronts of 128 rows x 64 columns, two to a SIMD: TM = 256 is one workgroup of eight per CU, TM = 128 two of four.
template <int TM>
__global__ void __launch_bounds__(TM * 2, 2) k_expert_dw(DwMulti m) {
  constexpr int kWaves = TM / 32, kRowA = TM * 2, kBytesA = TK * kRowA, kStage = kBytesA + kBytesB;
  constexpr int kPiecesA = kBytesA / 1024 / kWaves, kPiecesB = kBytesB / 1024 / kWaves, kPieces = kPiecesA + kPiecesB;
  static_assert(kWaves * 8192 <= kStages * kStage, "room for the way out");
  __shared__ __attribute__((aligned(1024))) unsigned char ring[kStages * kStage];
  // Units of some tiles of one weight go round the XCDs, back and forth: a unit's tiles read the same rows and share an L2, and with
  // the experts by falling length every XCD gets about as much.
  const int b = (int)blockIdx.x, xcd = b % kXcds, q = b / kXcds, round = q / m.unit;
  const int unit = round * kXcds + ((round & 1) ? kXcds - 1 - xcd : xcd), per = m.unit0[m.count], rank = unit / per, mine = unit - rank * per;
  if (rank >= m.experts) return;
  const int e = m.order[rank];
  if ((uint32_t)e >= (uint32_t)m.experts) return;
  int pi = 0;
  while (pi + 1 < m.count && mine >= m.unit0[pi + 1]) ++pi;
  const DwOne &p = m.p[pi];
  const int tile = (mine - m.unit0[pi]) * m.unit + q % m.unit;
  if (tile >= p.tiles) return;
  const int m0 = tile / p.tn * TM, n0 = (tile % p.tn) * TN;
  const int K = p.K, N = p.N, at = m.offsets[e], tokens = m.counts[e];
  const int64_t first = at < 0 ? 0 : at < m.capacity ? at : m.capacity, room = m.capacity - first;      // (a segment stays inside x and dy, whatever the arrays hold)
  const int rows = tokens < room ? tokens : (int)room;
  const int lane = (int)(threadIdx.x & 63), wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));

  Feed fa{(const char *)(p.x + first * K + m0), ((int64_t)rows * K - m0) * 2, (int64_t)TK * K * 2};
  Feed fb{(const char *)(p.dy + first * N + n0), ((int64_t)rows * N - n0) * 2, (int64_t)TK * N * 2};
  // Piece i of an operand's tile is 1 KiB of LDS: 4 rows of 256 bytes or 2 of 512. The 16-byte chunk of a row is XORed with 4 * (row & 3), so
  // that the four rows that a transposing read touches fall into different banks.
  uint32_t va[kPiecesA], vb[kPiecesB];
#pragma unroll
  for (int i = 0; i < kPiecesA; ++i) {
    const int row = (wave * kPiecesA + i) * (1024 / kRowA) + lane / (kRowA / 16);
    va[i] = (uint32_t)(row * K * 2 + (((lane % (kRowA / 16)) ^ ((row & 3) << 2)) * 16));
  }
#pragma unroll
  for (int i = 0; i < kPiecesB; ++i) {
    const int row = (wave * kPiecesB + i) * 2 + (lane >> 5);
    vb[i] = (uint32_t)(row * N * 2 + (((lane & 31) ^ ((row & 3) << 2)) * 16));
  }
  auto issue = [&](int i, const anc_i32x4 &da, const anc_i32x4 &db, unsigned char *stage) {
    if (i < kPiecesA) dma16_bounded(da, va[i], lds_addr(stage + (wave * kPiecesA + i) * 1024));
    else dma16_bounded(db, vb[i - kPiecesA], lds_addr(stage + kBytesA + (wave * kPiecesB + i - kPiecesA) * 1024));
  };
  auto issue_all = [&](unsigned char *stage) {
    const anc_i32x4 da = fa.desc(), db = fb.desc();
#pragma unroll
    for (int i = 0; i < kPieces; ++i) issue(i, da, db, stage);
    fa.next();
    fb.next();
  };

  // Fragments: lane -> column lane % 32 of a 32-column block, 8 consecutive tokens (8 * (lane / 32) on) of 16.
  int ta[4], tb[2];
  {
    const int s16 = lane & 15, g16 = lane >> 4, half = (s16 & 3) >> 1, row = 8 * (g16 >> 1) + (s16 >> 2), sw = (s16 >> 2) << 2;
#pragma unroll
    for (int i = 0; i < 4; ++i) ta[i] = row * kRowA + ((((wave >> 2) * 16 + i * 4 + 2 * (g16 & 1) + half) ^ sw) * 16) + (s16 & 1) * 8;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      tb[i] = kBytesA + row * kRowB + ((((wave & 3) * 8 + i * 4 + 2 * (g16 & 1) + half) ^ sw) * 16) + (s16 & 1) * 8;
  }
  f32x16 acc[4][2];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;

  const int steps = (rows + TK - 1) / TK;
  if (steps > 0) {
    bf16x8 a[2][4], c[2][2];
    // fragment i (0 .. 5: b0 b1 a0 a1 a2 a3) of 16 tokens kk of a stage
    auto load = [&](int set, int i, const unsigned char *stage, int kk) {
      if (i < 2) c[set][i] = anc_lds_tr_frag(stage + tb[i] + kk * (16 * 512), stage + tb[i] + kk * (16 * 512) + 4 * 512);
      else a[set][i - 2] = anc_lds_tr_frag(stage + ta[i - 2] + kk * (16 * kRowA), stage + ta[i - 2] + kk * (16 * kRowA) + 4 * kRowA);
    };
    auto multiply = [&](int set, int idx) {      // operands exchanged: a lane holds runs of 4 columns of one row
      acc[idx >> 1][idx & 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(c[set][idx & 1], a[set][idx >> 1], acc[idx >> 1][idx & 1], 0, 0, 0);
    };
    for (int i = 0; i < kStages; ++i) issue_all(ring + i * kStage);
    wait_vm<(kStages - 1) * kPieces>();
    lds_barrier();
#pragma unroll
    for (int i = 0; i < 6; ++i) load(0, i, ring, 0);
    // One step: the first half's products over the reads of the second half; then every wavefront has read the stage and the
    // next one has landed for all; then the second half's products over the next stage's first reads and the fetches of
    // the stage after the next two into the place just read.
    auto step = [&](unsigned char *here, unsigned char *next) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        multiply(0, i);
        __builtin_amdgcn_sched_barrier(0);
        if (i < 6) load(1, i, here, 1);
        __builtin_amdgcn_sched_barrier(0);
      }
      wait_vm<(kStages - 2) * kPieces>();
      lds_barrier();
      const anc_i32x4 da = fa.desc(), db = fb.desc();
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        multiply(1, i);
        __builtin_amdgcn_sched_barrier(0);
        if (i < 6) load(0, i, next, 0);
        if (i < kPieces) issue(i, da, db, here);
        __builtin_amdgcn_sched_barrier(0);
      }
      fa.next();
      fb.next();
    };
    int here = 0;
    for (int t = 0; t < steps; ++t) {
      const int next = here + kStage < kStages * kStage ? here + kStage : 0;
      step(ring + here, ring + next);
      here = next;
    }
  }
  wait_vm<0>();                                  // (zeros still on their way into the stages)
  lds_barrier();

  // Out through LDS, 32 rows of 64 columns at a time, so that stores are rows of 256 bytes.
  unsigned char *r = ring + wave * 8192;
  const int row0 = m0 + (wave >> 2) * 128;
  const int cols = N - n0 - (wave & 3) * 64;           // this wavefront's columns that exist
  const int64_t out0 = (int64_t)e * K * N + (int64_t)row0 * N + n0 + (wave & 3) * 64;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int rr = lane & 31, hh = lane >> 5;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *(anc_f32x4 *)(r + rr * 256 + (((j * 8 + 2 * g + hh) ^ (rr & 15)) * 16)) =
            anc_f32x4{acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
    lds_wave_sync();
#pragma unroll
    for (int z = 0; z < 8; ++z) {
      const int idx = z * 64 + lane, row = idx >> 4, ch = idx & 15;
      anc_f32x4 v = *(const anc_f32x4 *)(r + row * 256 + ((ch ^ (row & 15)) * 16));
      if (row0 + i * 32 + row < K && ch * 4 < cols) {
        const int64_t off = out0 + (int64_t)(i * 32 + row) * N + ch * 4;
        if (p.accumulate) {
          const anc_f32x4 o = *(const anc_f32x4 *)(p.dW + off);
          v = anc_f32x4{o.x + v.x, o.y + v.y, o.z + v.z, o.w + v.w};
        }
        anc_st_stream((anc_f32x4 *)(p.dW + off), v);
        if (p.g16 != nullptr) anc_st_stream((anc_u32x2 *)(p.g16 + off), anc_u32x2{anc_pk_bf16(v.x, v.y), anc_pk_bf16(v.z, v.w)});
      }
    }
    lds_wave_sync();
  }
}

}  // namespace

extern "C" int anc_expert_dw_multi(const anc_expert_dw_problem_t *probs, int32_t n_probs, uint64_t counts, uint64_t offsets,
                                   uint64_t order, int64_t experts, int64_t capacity, uint64_t stream) {
  ANC_REQUIRE(probs != nullptr && n_probs >= 1 && n_probs <= kMostProblems, "anc_expert_dw_multi: 1..%d problems", kMostProblems);
  ANC_REQUIRE(counts && offsets && order && ((counts | offsets | order) & 3) == 0 && experts > 0 && experts <= 512,
              "anc_expert_dw_multi: bad segments (%lld experts)", (long long)experts);
  ANC_REQUIRE(capacity > 0 && capacity < (1ll << 31), "anc_expert_dw_multi: room for %lld slots", (long long)capacity);
  DwMulti m{};
  m.capacity = capacity;
  m.counts = (const int32_t *)counts;
  m.offsets = (const int32_t *)offsets;
  m.order = (const int32_t *)order;
  m.count = n_probs;
  m.experts = (int)experts;
  int64_t wide = 0;                                  // tiles of 256x256
  AncSpan span[kMostProblems][4];                    // outputs, then inputs
  for (int i = 0; i < n_probs; ++i) {
    const anc_expert_dw_problem_t &b = probs[i];
    ANC_REQUIRE(b.K > 0 && b.N > 0 && b.K % 8 == 0 && b.N % 8 == 0 && b.K <= (1 << 17) && b.N <= (1 << 17),
                "anc_expert_dw_multi: needs K %% 8 == 0 and N %% 8 == 0 (K=%lld N=%lld)", (long long)b.K, (long long)b.N);
    ANC_REQUIRE(b.x && b.dy && b.dW && ((b.x | b.dy | b.dW) & 15) == 0 && (b.g16 & 7) == 0,
                "anc_expert_dw_multi: null or misaligned pointer");
    span[i][0] = {b.dW, experts * b.K * b.N * 4};
    span[i][1] = {b.g16, b.g16 != 0 ? experts * b.K * b.N * 2 : 0};
    span[i][2] = {b.x, capacity * b.K * 2};
    span[i][3] = {b.dy, capacity * b.N * 2};
    m.p[i] = DwOne{(const uint16_t *)b.x, (const uint16_t *)b.dy, (float *)b.dW, (uint16_t *)b.g16, (int)b.K, (int)b.N,
                   (int)((b.N + TN - 1) / TN), 0, b.accumulate != 0};
    wide += (b.K + 255) / 256 * m.p[i].tn * experts;
  }
  for (int i = 0; i < n_probs; ++i)                  // (workgroups run in any order: an output meets no other buffer of the call)
    for (int a = 0; a < 2; ++a)
      for (int j = 0; j < n_probs; ++j)
        for (int c = 0; c < 4; ++c)
          ANC_REQUIRE((i == j && a == c) || anc_apart(span[i][a].at, span[i][a].bytes, span[j][c].at, span[j][c].bytes),
                      "anc_expert_dw_multi: an output of problem %d overlaps a buffer of problem %d", i, j);
  for (int i = 0; i < n_probs; ++i)
    ANC_REQUIRE(anc_outputs_apart({span[i][0], span[i][1], {counts, 4 * experts}, {offsets, 4 * experts + 4}, {order, 4 * experts}}, 2),
                "anc_expert_dw_multi: an output of problem %d overlaps the segments", i);
  // 256x256 tiles where they give every CU one and there is room for 256 rows per expert: fewer operand bytes for a product. With fewer
  // tiles twice as many of 128x256 are at work; with short segments the two workgroups of a CU hide each other's ends. Room is what
  // the host knows: filling, tokens without an expert and tokens that the plan could hold count in it, so that segments may be much shorter
  // than the line says, and around the line the better side hangs on the shape and on what is cached. A layer's three weights with bf16 copies
  // and its five operands, us, 256x256 and 128x256: 16 experts of 1024x1024 with 1024 rows each 147 and 155, 768 125 and 134, 512 99 and 92 (with
  // operands of each weight's own 102 and 114), 256 79 and 72, 128 68 and 63, 64 filled up to 256 62 and 60; 64 experts of 512x1024 with
  // 512 rows 208 and 219, 256 168 and 182, 128 filled up to 256 135 and 132; 128 experts of 512x768 with 256 rows 265 and 249; 8 experts, one weight
  // of 512x512, 512 rows 19.0 and 14.5.
  const int TM = wide >= 256 && capacity >= 256 * experts ? 256 : 128;
  for (int i = 0; i < n_probs; ++i) m.p[i].tiles = (m.p[i].K + TM - 1) / TM * m.p[i].tn;
  // The tiles that stay together: a whole weight of 16 or 32 tiles, fewer where that leaves an XCD less than six units to even out.
  for (m.unit = 32;; m.unit /= 2) {
    m.unit0[0] = 0;
    for (int i = 0; i < n_probs; ++i) m.unit0[i + 1] = m.unit0[i] + (m.p[i].tiles + m.unit - 1) / m.unit;
    if (m.unit == 4 || m.unit0[n_probs] * experts >= 6 * kXcds) break;
  }
  const int64_t units = m.unit0[n_probs] * experts, grid = (units + kXcds - 1) / kXcds * kXcds * m.unit;
  ANC_REQUIRE(grid * TM * 2 < (1ll << 32), "anc_expert_dw_multi: too large for one call");
  hipStream_t s = anc_stream(stream);
  AncProfScope prof(ANC_PROF_DW_GEMM, s);
  if (TM == 256) hipLaunchKernelGGL(k_expert_dw<256>, dim3((unsigned)grid), dim3(512), 0, s, m);
  else           hipLaunchKernelGGL(k_expert_dw<128>, dim3((unsigned)grid), dim3(256), 0, s, m);
  ANC_LAUNCH_CHECK();
  return ANC_OK;
}
