// Small integer keys put in order on the device: token ids into groups of one id, (token, choice) assignments into
// segments of one expert. Both are a stable sort, so that what is summed up over a group is summed in the tokens' order
// and the same on every run.
//
// Ranking: a wavefront takes 64 consecutive items at a time. The lanes that hold the same digit are found with one ballot
// per bit of the digit; an item's rank is the number of earlier lanes among them plus the wavefront's count of the digit
// so far, a counter in LDS. Items of different wavefronts meet in an exclusive sum over (digit, wavefront).
//
// Ids of up to kMostSplit positions are grouped in one launch: every workgroup looks at all ids, takes those of its share of the order
// (shares cut by a sample), sorts them in LDS and writes them where they belong; what lies before its share it has counted on the
// way. A launch costs as much as looking at some ten thousand ids. Beyond, passes of 9 bits over blocks of kBlock items with the
// blocks' digit counts in memory: a block adds up the counts before it itself (no launch in between), and the count for the next pass is
// made by the scatter, with integer atomics, which have no order to lose.
#include "common.h"

namespace {

typedef int anc_i32x4 __attribute__((ext_vector_type(4)));

constexpr int kDigitBits = 9, kDigits = 1 << kDigitBits;
constexpr int kBlockLanes = 256, kBlockItems = 8, kBlock = kBlockLanes * kBlockItems;

// Lanes of the wavefront that hold the same digit as this one, among those with `in`. (Six vector instructions a bit: the digit's bit
// as 0 or -1, its ballot, and two words of agreement.)
__device__ __forceinline__ uint64_t same_digit(uint32_t d, int bits, bool in) {
  const uint64_t all = __ballot(in);
  const int first = all != 0 ? __builtin_ctzll(all) : 0;
  if (__ballot(in && d == (uint32_t)__builtin_amdgcn_readlane((int)d, first)) == all) return all;      // (a frequent id's run)
  uint32_t lo = (uint32_t)all, hi = (uint32_t)(all >> 32);
  for (int b = 0; b < bits; ++b) {
    const uint32_t s = (uint32_t)__builtin_amdgcn_sbfe((int)d, b, 1);
    const uint64_t v = __ballot(s != 0);
    lo &= ~((uint32_t)v ^ s);
    hi &= ~((uint32_t)(v >> 32) ^ s);
  }
  return (uint64_t)hi << 32 | lo;
}
__device__ __forceinline__ int lanes_before(uint64_t m) {
  return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
}
// Rank of this lane's item among the wavefront's items of its digit so far; `count` is the wavefront's own row in LDS. Lanes without
// `in` take no part.
__device__ __forceinline__ int take_rank(volatile int *count, uint32_t d, int bits, bool in) {
  const uint64_t m = same_digit(d, bits, in);
  const int before = lanes_before(m);
  int old = 0;
  if (in) old = count[d];
  __builtin_amdgcn_wave_barrier();
  if (in && before == 0) count[d] = old + __popcll(m);
  __builtin_amdgcn_wave_barrier();
  return old + before;
}
// Sums across lanes within registers: DPP moves feed the addition itself (through LDS a step is some hundred clocks: the three
// sums of a grouping of 8192 ids took 2.3 us).
__device__ __forceinline__ int wave_scan(int v) {          // inclusive
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);      // from 1, 2, 4, 8 lanes below, within 16
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);      // lane 15 of a row of 16 to the next row, rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);      // lane 31 to rows 2 and 3
  return v;
}
__device__ __forceinline__ int wave_sum(int v) { return __builtin_amdgcn_readlane(wave_scan(v), 63); }
template <int L> __device__ __forceinline__ int sum_of(int v) {        // over L neighbours
  static_assert(L == 1 || L == 2 || L == 4, "within four lanes");
  if constexpr (L >= 2) v += __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xF, 0xF, true);         // lanes 1 0 3 2
  if constexpr (L == 4) v += __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xF, 0xF, true);         // lanes 2 3 0 1
  return v;
}
// Exclusive sum over the workgroup's lanes, in lane order; every lane calls. total: the sum over all.
template <int LANES>
__device__ __forceinline__ int block_scan(int v, int *tmp, int &total) {
  constexpr int W = LANES / 64;
  const int wave = (int)(threadIdx.x >> 6), lane = (int)(threadIdx.x & 63);
  const int inc = wave_scan(v);
  __syncthreads();                                    // (tmp may still be read from before)
  if (lane == 63) tmp[wave] = inc;
  __syncthreads();
  int base = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    const int t = tmp[w];
    base += w < wave ? t : 0;
    total += t;
  }
  total = __builtin_amdgcn_readfirstlane(total);
  return base + inc - v;
}

// The ids at `first`, first + step, ..., as keys: V for one that names no row and for what lies behind the last. (Addresses are
// clamped instead of the loads guarded, so that all of them are in flight at once; n > 0.)
template <int ITEMS>
__device__ __forceinline__ void load_keys(const void *ids, int wide, int64_t first, int step, int64_t n, uint32_t V, uint32_t (&key)[ITEMS]) {
  int64_t id[ITEMS];
  if (wide) {
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
      const int64_t p = first + (int64_t)j * step;
      id[j] = ((const int64_t *)ids)[p < n ? p : n - 1];
    }
  } else {
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
      const int64_t p = first + (int64_t)j * step;
      id[j] = ((const int32_t *)ids)[p < n ? p : n - 1];
    }
  }
#pragma unroll
  for (int j = 0; j < ITEMS; ++j)
    key[j] = first + (int64_t)j * step < n && id[j] >= 0 && id[j] < (int64_t)V ? (uint32_t)id[j] : V;
}

struct Groups {
  int32_t *srt, *start, *cnt, *gid;                  // as build_id_groups lays them out, M long
  int32_t *key, *grp;                                // id and group of every sorted position (V, -1: names no row)
  int32_t *count;                                    // number of groups
};

// ---------------------------------------------------------------- token ids, one launch
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
// An item's place in the order, as a number: its id, then its position.
__device__ __forceinline__ uint64_t place(uint32_t key, int p) { return (uint64_t)key << 32 | (uint32_t)p; }
// A token id as a key: V for one that names no row.
__device__ __forceinline__ uint32_t as_key(int32_t id, uint32_t V) { return (uint32_t)id < V ? (uint32_t)id : V; }
__device__ __forceinline__ uint32_t as_key(int64_t id, uint32_t V) { return (uint64_t)id < V ? (uint32_t)id : V; }
constexpr int kPartItems = 4, kSamples = 256;
// Both sides measured, ids of 152 K rows, a call in a row of calls: 512 alone on 256 lanes 7.0 us (on 1024 7.7), 1024 alone on 512 lanes 7.5 (on
// 1024 8.4; in shares 9.2), 1500 alone 8.8, 2048 alone 10.2 and in shares 9.3; shares on 512 and on 1024 lanes: 8192 12.4 and 13.8, 24000 20.1 and
// 20.8, 32768 23.2 and 23.0; 65536 in shares 31, by passes 47. Where a table has more rows than bits in LDS the passes are all there is: 2^18
// rows and one more, 1537 ids 10 and 34 us, 8192 13 and 52, 65536 32 and 73; beyond 65536 ids 131072 take 52 (2 passes) and 82 (3), 2^20 143 and 227.
constexpr int64_t kFewAlone = 512, kMostAlone = 1536, kFewSplit = 1 << 14, kMostSplit = 1 << 16;             // positions: of one workgroup, of several
constexpr int64_t kMostMarked = 1 << 18;                               // ids, where several workgroups share them (one bit each in LDS)

// SPLIT: gridDim.x workgroups share the order; else one takes all of it (n <= CAP, and any V).
template <int LANES, bool SPLIT, typename ID>
__global__ void __launch_bounds__(LANES)
k_group_part(const ID *__restrict__ ids, int n, int64_t M, uint32_t V, Groups o) {
  constexpr int W = LANES / 64, CAP = LANES * kPartItems, PER = kDigits > LANES ? kDigits / LANES : 1, kTile = 8;
  __shared__ uint32_t skey[CAP];
  __shared__ int spos[SPLIT ? CAP : 1];
  __shared__ uint16_t sidx[CAP];
  __shared__ __attribute__((aligned(16))) int count[W * kDigits];      // (also the sample, and where the groups begin)
  __shared__ int tmp[W];
  __shared__ anc_i32x4 four[W];
  __shared__ int cut[4];
  __shared__ uint32_t last_id;
  __shared__ uint32_t marks[SPLIT ? kMostMarked / 32 : 1];
  static_assert(W * kDigits >= CAP && W * kDigits >= kSamples, "count is used three ways");
  const int tid = (int)threadIdx.x, wave = uniform(tid >> 6), lane = tid & 63, parts = (int)gridDim.x, part = (int)blockIdx.x;
  uint32_t id_lo = 0, id_hi = V + 1;                 // this workgroup's share: from (id_lo, p_lo) to (id_hi, p_hi)
  int p_lo = 0, p_hi = 0;
  const int words = (int)((V + 31) / 32);
  // A wavefront looks at `share` positions next to each other (64 times 64 at most), kTile times 64 at a time.
  const int share = ((n + W - 1) / W + 63) / 64 * 64, w0 = wave * share, w1 = w0 + share < n ? w0 + share : n;
  uint32_t key[kTile];
  ID raw[kTile];
  auto fetch = [&](int t) {
#pragma unroll
    for (int j = 0; j < kTile; ++j) raw[j] = ids[t + 64 * j + lane < w1 ? t + 64 * j + lane : w1 - 1];
  };
  // f(a tile's first position) for all tiles of the wavefront, its keys there, the next tile's ids on their way.
  bool ready = true;
  auto each_tile = [&](auto f) {
    if (!ready && w0 < w1) fetch(w0);
    ready = false;
#pragma unroll 1
    for (int t = w0; t < w1; t += 64 * kTile) {
#pragma unroll
      for (int j = 0; j < kTile; ++j) key[j] = as_key(raw[j], V);
      if (t + 64 * kTile < w1) fetch(t + 64 * kTile);
      f(t);
    }
  };
  if (w0 < w1) fetch(w0);
  if constexpr (SPLIT) {
    // Every workgroup sorts the same sample, a position of every n / kSamples, spread by a multiplicative hash, by looking at all of it, and
    // cuts the order at its own two of the shares.
    constexpr int L = LANES / kSamples;              // lanes per sample, neighbours, each looking at a run of the others
    uint32_t *sample = (uint32_t *)count;
    const int i = tid / L, at = (int)((int64_t)i * n / kSamples) + (int)(((uint32_t)i * 2654435761u >> 8) % (uint32_t)(n / kSamples));
    const uint32_t id = as_key(ids[at], V), mine = id << 8 | (uint32_t)i;  // (at most 19 bits of id, and the sample's own order)
    for (int w = tid; w < words; w += LANES) marks[w] = 0;
    if (tid % L == 0) sample[i] = mine;
    if (tid < 4) cut[tid] = tid == 2 ? (int)(V + 1) : 0;
    __syncthreads();
    int before = 0;
    const anc_u32x4 *run = (const anc_u32x4 *)sample + (tid % L) * (kSamples / L / 4);
#pragma unroll
    for (int j = 0; j < kSamples / L / 4; ++j) {
      const anc_u32x4 v = run[j];
      before += (v.x < mine ? 1 : 0) + (v.y < mine ? 1 : 0) + (v.z < mine ? 1 : 0) + (v.w < mine ? 1 : 0);
    }
    before = sum_of<L>(before);
    if (tid % L == 0) {
      if (part > 0 && before == part * kSamples / parts) { cut[0] = (int)id; cut[1] = at; }
      if (part + 1 < parts && before == (part + 1) * kSamples / parts) { cut[2] = (int)id; cut[3] = at; }
    }
    __syncthreads();
    id_lo = (uint32_t)uniform(cut[0]);
    p_lo = uniform(cut[1]);
    id_hi = (uint32_t)uniform(cut[2]);
    p_hi = uniform(cut[3]);
  }
  bool marked = false;
  int groups = 0;                                    // of the whole batch
  while (place(id_lo, p_lo) < place(id_hi, p_hi)) {
    uint32_t id_to = id_hi;                          // the piece that is done at once ends at (id_to, p_to)
    uint64_t mask = 0;
    int p_to = p_hi, size = n, put = 0, base = 0, came = 0, goes = 0, smaller = 0;
    if constexpr (SPLIT) {
      const uint64_t lo = place(id_lo, p_lo);
      for (;;) {
        // Lane i keeps which of the wavefront's i-th 64 positions belong to the piece. Counted are the items before it, those of its first
        // id before it and those of the id it ends in behind it.
        const uint64_t to = place(id_to, p_to);
        mask = 0;
        int low = 0, came_goes = 0;                  // (of a lane, then of a wavefront: at most 64 and 4096)
        each_tile([&](int t) {
          // (Lanes that meet on a word take turns: of a run of one id its first lane goes, of an id that is frequent everywhere, padding, the
          // wavefront's first. 65536 ids in runs of 16: 33 us; with every item reading first whether its bit is set 67.)
          if (!marked) {
#pragma unroll
            for (int j = 0; j < kTile; ++j) {
              const uint32_t left = (uint32_t)__builtin_amdgcn_update_dpp((int)V, (int)key[j], 0x138, 0xF, 0xF, false);
              const uint32_t of_lane0 = (uint32_t)uniform((int)key[j]);          // (read while every lane is active)
              if (key[j] < V && key[j] != left && (lane == 0 || key[j] != of_lane0)) atomicOr(&marks[key[j] >> 5], 1u << (key[j] & 31));
            }
          }
#pragma unroll
          for (int j = 0; j < kTile; ++j) {
            if (t + 64 * j >= w1) break;
            const int p = t + 64 * j + lane;
            const uint64_t r = place(key[j], p);
            const bool there = p < w1, is_low = r < lo, is_high = r >= to;
            const uint64_t m = __ballot(there && !is_low && !is_high);
            if (lane == (t - w0) / 64 + j) mask = m;
            low += there && is_low ? 1 : 0;
            if (__ballot(key[j] == id_lo || key[j] == id_to) != 0)
              came_goes += there && is_low && key[j] == id_lo ? 1 : there && is_high && key[j] == id_to ? 0x10000 : 0;
          }
        });
        marked = true;
        const int own = __popcll(mask), upto = wave_scan(own);
        low = wave_sum(low);
        came_goes = wave_sum(came_goes);
        if (lane == 63) four[wave] = anc_i32x4{upto, low, came_goes & 0xFFFF, came_goes >> 16};
        __syncthreads();
        anc_i32x4 sum = {0, 0, 0, 0};
        put = upto - own;                            // this lane's first
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const anc_i32x4 v = four[w];
          put += w < wave ? v.x : 0;
          sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
        }
        size = uniform(sum.x);
        base = uniform(sum.y);
        came = uniform(sum.z);
        goes = uniform(sum.w);
        __syncthreads();
        if (size <= CAP) break;
        // More than LDS holds: the largest beginning that fits, by some 50 more looks at all ids. On average a share is a sixteenth (512
        // lanes) or an eighth of that, and it spans two samples: of 65536 mostly distinct ids one call in some 6000 meets such a share, of
        // 50000 one in a million. Where the sample sees nothing of the order (all sampled positions on one id) 8192 ids take 170 us, 20000 530,
        // 65536 4800.
        uint64_t fits = lo, over = to;
        while (over - fits > 1) {
          const uint64_t mid = fits + (over - fits) / 2;
          int some = 0, total;
          each_tile([&](int t) {
#pragma unroll
            for (int j = 0; j < kTile; ++j) {
              const uint64_t r = place(key[j], t + 64 * j + lane);
              some += t + 64 * j + lane < w1 && r >= lo && r < mid ? 1 : 0;
            }
          });
          block_scan<LANES>(some, tmp, total);
          if (total <= CAP) fits = mid; else over = mid;
        }
        id_to = (uint32_t)(fits >> 32);
        p_to = (int)(uint32_t)fits;
      }
      // Ids below the piece's first, and all of them << 16. A wavefront counts at most 2^14: on 1024 lanes its part of the words holds no
      // more bits, on 512 the batch has no more ids.
      static_assert(kMostMarked / W <= 1 << 14 || (LANES == 512 && kFewSplit <= 1 << 14), "two sums in a word");
      int low_every = 0;
      for (int i = tid; i < words; i += LANES) {
        const uint32_t w = marks[i], i32 = (uint32_t)i * 32;
        low_every += __popc(w) << 16 | (i32 + 32 <= id_lo ? __popc(w) : i32 >= id_lo ? 0 : __popc(w & ((1u << (id_lo - i32)) - 1)));
      }
      low_every = wave_sum(low_every);
      if (lane == 0) tmp[wave] = low_every;
      for (; mask != 0; mask &= mask - 1) spos[put++] = w0 + lane * 64 + (int)__builtin_ctzll(mask);
      __syncthreads();
#pragma unroll
      for (int j = 0; j < kPartItems; ++j)
        if (tid + j * LANES < size) skey[tid + j * LANES] = as_key(ids[spos[tid + j * LANES]], V);
      groups = 0;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        smaller += tmp[w] & 0xFFFF;
        groups += (int)((uint32_t)tmp[w] >> 16);
      }
      smaller = uniform(smaller);
      groups = uniform(groups);
      __syncthreads();
    } else {
      each_tile([&](int t) {
#pragma unroll
        for (int j = 0; j < kTile; ++j)
          if (t + 64 * j + lane < w1) skey[t + 64 * j + lane] = key[j];
      });
      __syncthreads();
    }
    // The piece by its ids, relative to the first. Up to RANKED items are counted against each other: an item's rank is the number of smaller
    // (id, place in the piece), L lanes look for it. More go by up to 9 bits a pass. `items` per lane, a wavefront's next to each other.
    const int items = (size + LANES - 1) / LANES, first = wave * 64 * items + lane;
    const int bits = 32 - __builtin_clz((id_to - id_lo) | 1);
    const int passes = (bits + kDigitBits - 1) / kDigitBits, per = (bits + passes - 1) / passes;
    int idx[kPartItems], rank[kPartItems];
    uint32_t k[kPartItems];
#pragma unroll
    for (int j = 0; j < kPartItems; ++j) {
      idx[j] = first + 64 * j;
      k[j] = j < items && idx[j] < size ? skey[idx[j]] : 0;
    }
    constexpr int RANKED = LANES < 512 ? LANES : 512, L = LANES / RANKED;
    const bool by_rank = size <= RANKED && bits <= 22;
    if (by_rank) {
      uint32_t *numbers = (uint32_t *)count;
      if (tid < RANKED) numbers[tid] = tid < size ? (k[0] - id_lo) << 9 | (uint32_t)tid : ~0u;
      __syncthreads();
      const uint32_t mine = numbers[tid / L];
      int smaller_ones = 0;
      for (int v = tid % L; v * 4 < size; v += L) {
        const anc_u32x4 q = ((const anc_u32x4 *)numbers)[v];
        smaller_ones += (q.x < mine ? 1 : 0) + (q.y < mine ? 1 : 0) + (q.z < mine ? 1 : 0) + (q.w < mine ? 1 : 0);
      }
      smaller_ones = sum_of<L>(smaller_ones);
      if (tid % L == 0 && tid / L < size) sidx[smaller_ones] = (uint16_t)(tid / L);
      __syncthreads();
      if (tid < size) {
        idx[0] = sidx[tid];
        k[0] = skey[idx[0]];
      }
    }
    for (int shift = by_rank ? bits : 0; shift < bits; shift += per) {
      const int b = bits - shift < per ? bits - shift : per, digits = 1 << b;
      for (int i = tid; i < W << b; i += LANES) count[i] = 0;
      __syncthreads();
#pragma unroll
      for (int j = 0; j < kPartItems; ++j)
        if (j < items) rank[j] = take_rank(count + (wave << b), ((k[j] - id_lo) >> shift) & (digits - 1), b, first + 64 * j < size);
      __syncthreads();
      int c[PER][W], sum = 0, total;                 // PER digits of a lane, next to each other
#pragma unroll
      for (int q = 0; q < PER; ++q)
#pragma unroll
        for (int w = 0; w < W; ++w) {
          c[q][w] = tid * PER + q < digits ? count[(w << b) + tid * PER + q] : 0;
          sum += c[q][w];
        }
      int at = block_scan<LANES>(sum, tmp, total);
#pragma unroll
      for (int q = 0; q < PER; ++q)
        if (tid * PER + q < digits) {
#pragma unroll
          for (int w = 0; w < W; ++w) {
            count[(w << b) + tid * PER + q] = at;
            at += c[q][w];
          }
        }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < kPartItems; ++j)
        if (j < items && first + 64 * j < size)
          sidx[count[(wave << b) + (((k[j] - id_lo) >> shift) & (digits - 1))] + rank[j]] = (uint16_t)idx[j];
      __syncthreads();
#pragma unroll
      for (int j = 0; j < kPartItems; ++j)
        if (j < items && first + 64 * j < size) {
          idx[j] = sidx[first + 64 * j];
          k[j] = skey[idx[j]];
        }
    }
    // Heads: the first item of an id. Their number up to an item is its group, counted from the ids below the piece.
    int heads = 0, mine = 0, valid = 0;
#pragma unroll
    for (int j = 0; j < kPartItems; ++j) {
      const int p = first + 64 * j;
      if (j >= items || p >= size) continue;
      const bool head = k[j] < V && (p == 0 ? came == 0 || k[j] != id_lo : skey[sidx[p - 1]] != k[j]);
      heads |= head ? 1 << j : 0;
      mine += head ? 1 : 0;
      valid += k[j] < V ? 1 : 0;
    }
    int both;                                        // heads and items that name a row (CAP at most)
    int run = uniform(block_scan<LANES>(mine | valid << 16, tmp, both)) & 0xFFFF;        // (lane 0's: heads of the wavefronts before this one)
    const int n_heads = both & 0xFFFF, n_valid = both >> 16;
    const int group0 = smaller + (came > 0 && id_lo < V ? 1 : 0);
#pragma unroll
    for (int j = 0; j < kPartItems; ++j) {
      const int p = first + 64 * j;
      const bool head = (heads >> j) & 1;
      const uint64_t m = __ballot(head);
      const int h = run + lanes_before(m) + (head ? 1 : 0);
      run += __popcll(m);
      if (j >= items || p >= size) continue;
      const int g = group0 + h - 1;
      o.srt[base + p] = SPLIT ? spos[idx[j]] : idx[j];
      o.key[base + p] = (int32_t)k[j];
      o.grp[base + p] = k[j] < V ? g : -1;
      if (head) {
        count[h - 1] = p;
        if (h == n_heads) last_id = k[j];
        o.start[g] = base + p;
        o.gid[g] = (int32_t)k[j];
      }
    }
    __syncthreads();
    for (int h = tid; h < n_heads; h += LANES)       // (the last group may go on behind the piece)
      o.cnt[group0 + h] = (h + 1 < n_heads ? count[h + 1] : n_valid + (last_id == id_to ? goes : 0)) - count[h];
    if constexpr (!SPLIT) groups = n_heads;
    __syncthreads();
    id_lo = id_to;
    p_lo = p_to;
  }
  for (int64_t g = groups + (int64_t)part * LANES + tid; g < M; g += (int64_t)parts * LANES) {
    o.start[g] = 0;
    o.cnt[g] = 0;
    o.gid[g] = -1;
  }
  if (part == 0 && tid == 0) *o.count = groups;
}

// ---------------------------------------------------------------- token ids, many workgroups
// Digit counts of the first pass; what later passes and the groups count up is cleared.
__global__ void __launch_bounds__(kBlockLanes)
k_radix_count(const void *__restrict__ ids, int wide, int64_t n, int64_t M, uint32_t V, int bits, int passes,
              int *__restrict__ hist, int32_t *__restrict__ cnt) {
  __shared__ int h[kDigits];
  const int tid = (int)threadIdx.x;
  const int64_t blocks = gridDim.x, b = blockIdx.x;
  uint32_t key[kBlockItems];
  load_keys<kBlockItems>(ids, wide, b * kBlock + tid, kBlockLanes, n, V, key);
  for (int i = tid; i < kDigits; i += kBlockLanes) h[i] = 0;
  __syncthreads();
  const uint32_t mask = bits < kDigitBits ? (1u << bits) - 1 : (uint32_t)kDigits - 1;
#pragma unroll
  for (int j = 0; j < kBlockItems; ++j)
    if (b * kBlock + j * kBlockLanes + tid < n) atomicAdd(&h[key[j] & mask], 1);
  __syncthreads();
  for (int i = tid; i < kDigits; i += kBlockLanes) {
    hist[b * kDigits + i] = h[i];
    for (int q = 1; q < passes; ++q) hist[(q * blocks + b) * kDigits + i] = 0;
  }
  for (int64_t i = b * kBlockLanes + tid; i < M; i += blocks * kBlockLanes) cnt[i] = 0;
}

// One stable pass over bits shift .. of the keys.
__global__ void __launch_bounds__(kBlockLanes)
k_radix_scatter(const void *__restrict__ ids, int wide, const int32_t *__restrict__ key_in,
                const int32_t *__restrict__ idx_in, int64_t n, uint32_t V, int shift, int bits,
                const int *__restrict__ hist, int *__restrict__ hist_next, int32_t *__restrict__ key_out,
                int32_t *__restrict__ idx_out) {
  constexpr int W = kBlockLanes / 64, PER = kDigits / kBlockLanes;
  __shared__ int count[W * kDigits];
  __shared__ int tmp[W];
  const int tid = (int)threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int64_t blocks = gridDim.x, b = blockIdx.x, first = b * kBlock + wave * (64 * kBlockItems) + lane;
  const int nb = bits - shift < kDigitBits ? bits - shift : kDigitBits;
  const uint32_t mask = (1u << nb) - 1;
  uint32_t key[kBlockItems];
  int32_t idx[kBlockItems];
  if (key_in != nullptr) {
#pragma unroll
    for (int j = 0; j < kBlockItems; ++j) {
      const int64_t p = first + 64 * j < n ? first + 64 * j : n - 1;
      key[j] = (uint32_t)key_in[p];
      idx[j] = idx_in[p];
    }
  } else {
    load_keys<kBlockItems>(ids, wide, first, 64, n, V, key);
#pragma unroll
    for (int j = 0; j < kBlockItems; ++j) idx[j] = (int32_t)(first + 64 * j);
  }
  for (int i = tid; i < W * kDigits; i += kBlockLanes) count[i] = 0;
  // counts of this lane's digits over all blocks, and over the blocks before this one
  int all[PER], below[PER];
#pragma unroll
  for (int q = 0; q < PER; ++q) all[q] = below[q] = 0;
  constexpr int D = 16;
  for (int64_t c = 0; c < blocks; c += D) {
    int v[D][PER];
#pragma unroll
    for (int i = 0; i < D; ++i)
#pragma unroll
      for (int q = 0; q < PER; ++q) v[i][q] = hist[(c + i < blocks ? c + i : blocks - 1) * kDigits + tid * PER + q];
#pragma unroll
    for (int i = 0; i < D; ++i)
#pragma unroll
      for (int q = 0; q < PER; ++q) {
        all[q] += c + i < blocks ? v[i][q] : 0;
        below[q] += c + i < b ? v[i][q] : 0;
      }
  }
  __syncthreads();
  int rank[kBlockItems];
#pragma unroll
  for (int j = 0; j < kBlockItems; ++j)
    rank[j] = take_rank(count + wave * kDigits, (key[j] >> shift) & mask, nb, first + 64 * j < n);
  int sum = 0, total;
#pragma unroll
  for (int q = 0; q < PER; ++q) sum += all[q];
  int base = block_scan<kBlockLanes>(sum, tmp, total);       // (its barriers also end the ranking)
#pragma unroll
  for (int q = 0; q < PER; ++q) {
    int at = base + below[q];
    base += all[q];
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const int c = count[w * kDigits + tid * PER + q];
      count[w * kDigits + tid * PER + q] = at;
      at += c;
    }
  }
  __syncthreads();
  // The next pass's digit counts, by the blocks that the items move to. One atomic for the lanes that agree in both (a frequent id
  // is thousands of items of one block and digit), one each for the few whose neighbours went to another block.
  const int left = bits - shift - kDigitBits, next_bits = left < kDigitBits ? left : kDigitBits;
#pragma unroll
  for (int j = 0; j < kBlockItems; ++j) {
    const bool in = first + 64 * j < n;
    const int at = in ? count[wave * kDigits + ((key[j] >> shift) & mask)] + rank[j] : 0;
    if (in) {
      key_out[at] = (int32_t)key[j];
      idx_out[at] = idx[j];
    }
    if (hist_next != nullptr) {
      const uint32_t next = (key[j] >> (shift + kDigitBits)) & ((1u << next_bits) - 1);
      const int to = at / kBlock;
      const uint64_t same = same_digit(next, next_bits, in);
      const int leader = in ? __builtin_ctzll(same) : lane, to_leader = __shfl(to, leader, 64);
      const uint64_t with = same & __ballot(to == to_leader);
      if (in && (lane == leader || to != to_leader))
        atomicAdd(&hist_next[(int64_t)to * kDigits + next], lane == leader ? __popcll(with) : 1);
    }
  }
}

// Bit j: item first + j * step begins a group.
__device__ __forceinline__ int head_bits(const int32_t *key, int64_t first, int step, int64_t n, uint32_t V) {
  uint32_t k[kBlockItems], before[kBlockItems];
#pragma unroll
  for (int j = 0; j < kBlockItems; ++j) {
    const int64_t p = first + (int64_t)j * step < n ? first + (int64_t)j * step : n - 1;
    k[j] = (uint32_t)key[p];
    before[j] = (uint32_t)key[p > 0 ? p - 1 : 0];
  }
  int bits = 0;
#pragma unroll
  for (int j = 0; j < kBlockItems; ++j) {
    const int64_t p = first + (int64_t)j * step;
    bits |= p < n && k[j] < V && (p == 0 || before[j] != k[j]) ? 1 << j : 0;
  }
  return bits;
}
__global__ void __launch_bounds__(kBlockLanes)
k_heads(const int32_t *__restrict__ key, int64_t n, uint32_t V, int *__restrict__ heads) {
  __shared__ int tmp[kBlockLanes / 64];
  int total;
  block_scan<kBlockLanes>(__popc(head_bits(key, (int64_t)blockIdx.x * kBlock + threadIdx.x, kBlockLanes, n, V)), tmp, total);
  if (threadIdx.x == 0) heads[blockIdx.x] = total;
}
__global__ void __launch_bounds__(kBlockLanes)
k_groups(int64_t n, int64_t M, uint32_t V, const int *__restrict__ heads, Groups o) {
  __shared__ int tmp[kBlockLanes / 64];
  const int tid = (int)threadIdx.x, wave = tid >> 6, lane = tid & 63, blocks = (int)gridDim.x, b = (int)blockIdx.x;
  const int64_t first = (int64_t)b * kBlock + wave * (64 * kBlockItems) + lane;
  uint32_t k[kBlockItems], after[kBlockItems];
#pragma unroll
  for (int j = 0; j < kBlockItems; ++j) {
    const int64_t p = first + 64 * j < n ? first + 64 * j : n - 1;
    k[j] = (uint32_t)o.key[p];
    after[j] = (uint32_t)o.key[p + 1 < n ? p + 1 : p];
  }
  const int head = head_bits(o.key, first, 64, n, V);
  int all = 0, below = 0, total, run, in_block;
  for (int c = tid; c < blocks; c += kBlockLanes) {
    const int v = heads[c];
    all += v;
    below += c < b ? v : 0;
  }
  block_scan<kBlockLanes>(all, tmp, total);
  block_scan<kBlockLanes>(below, tmp, run);
  const int mine = __popc(head);
  run += block_scan<kBlockLanes>(mine, tmp, in_block) - (wave_scan(mine) - mine);
#pragma unroll
  for (int j = 0; j < kBlockItems; ++j) {
    const int64_t p = first + 64 * j;
    const bool is_head = (head >> j) & 1;
    const uint64_t m = __ballot(is_head);
    const int g = run + __popcll(m & ((1ull << lane) - 1)) - (is_head ? 0 : 1);
    run += __popcll(m);
    if (p >= n) continue;
    o.grp[p] = k[j] < V ? g : -1;
    if (is_head) {
      o.start[g] = (int32_t)p;
      o.gid[g] = (int32_t)k[j];
      atomicAdd(&o.cnt[g], -(int)p);                 // (a group's head and its last item meet in its count)
    }
    if (k[j] < V && (p + 1 == n || after[j] != k[j])) atomicAdd(&o.cnt[g], (int)p + 1);
  }
  for (int64_t g = total + (int64_t)b * kBlockLanes + tid; g < M; g += (int64_t)blocks * kBlockLanes) {
    o.start[g] = 0;
    o.gid[g] = -1;
  }
  if (b == 0 && tid == 0) *o.count = total;
}

// ---------------------------------------------------------------- assignments by expert
constexpr int kMostExperts = kDigits;

struct Route {
  int32_t *counts, *offsets, *order, *slot, *src;
};
// The experts by falling number of tokens, lower ones first where equal: an expert's place is the number of experts before it, found
// by looking at all of them (LANES / kMostOrdered lanes share the looking; behind the last expert scnt holds -1 up to a multiple of 4).
// Beyond kMostOrdered that would take longer than it gives: many short segments even out in any order.
constexpr int kMostOrdered = 256;
template <int LANES>
__device__ __forceinline__ void order_experts(const int *scnt, int E, int32_t *order) {
  if (E > kMostOrdered) {
    for (int e = (int)threadIdx.x; e < E; e += LANES) order[e] = e;
    return;
  }
  constexpr int L = LANES / kMostOrdered;            // lanes per expert, neighbours
  const int e = (int)threadIdx.x / L;
  const int mine = e < E ? scnt[e] : 0;
  int before = 0;
  for (int j = (int)threadIdx.x % L * 4; j < E; j += L * 4) {
    const anc_i32x4 c = *(const anc_i32x4 *)(scnt + j);
#pragma unroll
    for (int q = 0; q < 4; ++q) before += c[q] > mine || (c[q] == mine && j + q < e) ? 1 : 0;
  }
  before = sum_of<L>(before);
  if (e < E && (int)threadIdx.x % L == 0) order[before] = e;
}
__device__ __forceinline__ int filled_up(int c, int align) { return (c + align - 1) & -align; }

// Up to kMostCounted assignments in one launch: every workgroup counts all of them per expert, and those before its own, one to a lane, as the two
// halves of a word; four copies of the counters keep the lanes that meet on one apart.
// (16384 to 16 experts 6.3 us, two to a lane 7.0, counted and placed in two launches 9.9; 32768 8.5, 9.3 and 10.0)
constexpr int kMostCounted = 1 << 15, kOneLanes = 1024, kCopies = 4;
__global__ void __launch_bounds__(kOneLanes)
k_route_one(const void *__restrict__ ids, int wide, int n, int E, int bits, int align, int capacity, Route o) {
  constexpr int W = kOneLanes / 64;
  __shared__ int count[W * kMostExperts];
  __shared__ uint32_t hist[kCopies * kMostExperts];
  __shared__ int tmp[W];
  __shared__ int soff[kMostExperts + 1];
  __shared__ __attribute__((aligned(16))) int scnt[kMostExperts];
  const int tid = (int)threadIdx.x, wave = tid >> 6, lane = tid & 63, blocks = (int)gridDim.x, b = (int)blockIdx.x;
  const int p = b * kOneLanes + tid;
  uint32_t own[1] = {(uint32_t)E};                   // E: no expert
  if (n > 0) load_keys<1>(ids, wide, p, 0, n, (uint32_t)E, own);
  const uint32_t e = own[0];
  for (int i = tid; i < W * E; i += kOneLanes) count[i] = 0;
  for (int i = tid; i < kCopies * E; i += kOneLanes) hist[i] = 0;
  __syncthreads();
  constexpr int D = 8;
  for (int t = tid; blocks > 1 && t < n; t += D * kOneLanes) {
    uint32_t k[D];
    load_keys<D>(ids, wide, t, kOneLanes, n, (uint32_t)E, k);
#pragma unroll
    for (int j = 0; j < D; ++j)
      if (k[j] < (uint32_t)E) atomicAdd(&hist[k[j] * kCopies + (lane & (kCopies - 1))], t + j * kOneLanes < b * kOneLanes ? 0x10001u : 1u);
  }
  const int rank = take_rank(count + wave * E, e, bits, e < (uint32_t)E);
  __syncthreads();
  int all = 0, below = 0, c[W], total;
#pragma unroll
  for (int w = 0; w < W; ++w) c[w] = tid < E ? count[w * E + tid] : 0;
  if (blocks == 1) {
#pragma unroll
    for (int w = 0; w < W; ++w) all += c[w];
  } else if (tid < E) {
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      const uint32_t h = hist[tid * kCopies + i];
      all += (int)(h & 0xFFFF);
      below += (int)(h >> 16);
    }
  }
  const int base = block_scan<kOneLanes>(filled_up(all, align), tmp, total);
  if (tid < E) {
    int at = base + below;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      count[w * E + tid] = at;
      at += c[w];
    }
    soff[tid] = base;
    scnt[tid] = all;
    if (b == 0) { o.counts[tid] = all; o.offsets[tid] = base; }
  } else if (tid < kMostExperts) {
    scnt[tid] = -1;
  }
  if (tid == 0) {
    soff[E] = total;
    if (b == 0) o.offsets[E] = total;
  }
  __syncthreads();
  if (p < n) {
    const int s = e < (uint32_t)E ? count[wave * E + e] + rank : -1;
    o.slot[p] = s;
    if (s >= 0) o.src[s] = p;
  }
  if (b == blocks - 1) order_experts<kOneLanes>(scnt, E, o.order);
  for (int q = b * W + wave; q < E; q += blocks * W)
    for (int s = soff[q] + scnt[q] + lane; s < soff[q + 1]; s += 64) o.src[s] = -1;
  for (int64_t s = total + (int64_t)b * kOneLanes + tid; s < capacity; s += (int64_t)blocks * kOneLanes) o.src[s] = -1;
}

__global__ void __launch_bounds__(kBlockLanes)
k_route_count(const void *__restrict__ ids, int wide, int64_t n, int E, int *__restrict__ hist) {
  __shared__ int h[kMostExperts];
  const int tid = (int)threadIdx.x;
  uint32_t e[kBlockItems];
  load_keys<kBlockItems>(ids, wide, (int64_t)blockIdx.x * kBlock + tid, kBlockLanes, n, (uint32_t)E, e);
  for (int i = tid; i < E; i += kBlockLanes) h[i] = 0;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kBlockItems; ++j)
    if (e[j] < (uint32_t)E) atomicAdd(&h[e[j]], 1);
  __syncthreads();
  for (int i = tid; i < E; i += kBlockLanes) hist[(int64_t)blockIdx.x * E + i] = h[i];
}
__global__ void __launch_bounds__(kBlockLanes)
k_route_place(const void *__restrict__ ids, int wide, int64_t n, int E, int bits, int align, int64_t capacity,
              const int *__restrict__ hist, Route o) {
  constexpr int W = kBlockLanes / 64, PER = kMostExperts / kBlockLanes;
  __shared__ int count[W * kMostExperts];
  __shared__ int tmp[W];
  __shared__ int soff[kMostExperts + 1], sall[kMostExperts], sbelow[kMostExperts];
  __shared__ __attribute__((aligned(16))) int scnt[kMostExperts];
  const int tid = (int)threadIdx.x, wave = tid >> 6, lane = tid & 63, blocks = (int)gridDim.x, b = (int)blockIdx.x;
  const int64_t first = (int64_t)b * kBlock + wave * (64 * kBlockItems) + lane;
  uint32_t e[kBlockItems];
  int rank[kBlockItems], all[PER], below[PER];
  load_keys<kBlockItems>(ids, wide, first, 64, n, (uint32_t)E, e);
  for (int i = tid; i < W * E; i += kBlockLanes) count[i] = 0;
  // counts of every expert over all blocks and over the blocks before this one: `parts` lanes share an expert's column
  for (int i = tid; i < E; i += kBlockLanes) sall[i] = sbelow[i] = 0;
  __syncthreads();
  const int parts = E < kBlockLanes ? kBlockLanes / E : 1;
  for (int d = tid % E; d < E && tid < parts * E; d += kBlockLanes) {
    constexpr int D = 8;
    int a = 0, u = 0;
    for (int c = tid / E; c < blocks; c += D * parts) {
      int v[D];
#pragma unroll
      for (int i = 0; i < D; ++i) v[i] = hist[(int64_t)(c + i * parts < blocks ? c + i * parts : c) * E + d];
#pragma unroll
      for (int i = 0; i < D; ++i) {
        a += c + i * parts < blocks ? v[i] : 0;
        u += c + i * parts < b ? v[i] : 0;
      }
    }
    atomicAdd(&sall[d], a);
    atomicAdd(&sbelow[d], u);
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kBlockItems; ++j)
    rank[j] = take_rank(count + wave * E, e[j], bits, e[j] < (uint32_t)E);
  __syncthreads();
#pragma unroll
  for (int q = 0; q < PER; ++q) {
    const int d = tid * PER + q;
    all[q] = d < E ? sall[d] : 0;
    below[q] = d < E ? sbelow[d] : 0;
  }
  int sum = 0, total;
#pragma unroll
  for (int q = 0; q < PER; ++q) sum += filled_up(all[q], align);
  int base = block_scan<kBlockLanes>(sum, tmp, total);
#pragma unroll
  for (int q = 0; q < PER; ++q) {
    const int d = tid * PER + q;
    if (d < E) {
      soff[d] = base;
      scnt[d] = all[q];
      if (b == 0) { o.counts[d] = all[q]; o.offsets[d] = base; }
      int at = base + below[q];
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const int c = count[w * E + d];
        count[w * E + d] = at;
        at += c;
      }
    } else if (d < kMostExperts) {
      scnt[d] = -1;
    }
    base += filled_up(all[q], align);
  }
  if (tid == 0) {
    soff[E] = total;
    if (b == 0) o.offsets[E] = total;
  }
  __syncthreads();
  if (b == blocks - 1) order_experts<kBlockLanes>(scnt, E, o.order);
#pragma unroll
  for (int j = 0; j < kBlockItems; ++j) {
    const int64_t p = first + 64 * j;
    if (p >= n) continue;
    const int s = e[j] < (uint32_t)E ? count[wave * E + e[j]] + rank[j] : -1;
    o.slot[p] = s;
    if (s >= 0) o.src[s] = (int32_t)p;
  }
  for (int q = b * W + wave; q < E; q += blocks * W)
    for (int s = soff[q] + scnt[q] + lane; s < soff[q + 1]; s += 64) o.src[s] = -1;
  for (int64_t s = total + (int64_t)b * kBlockLanes + tid; s < capacity; s += (int64_t)blocks * kBlockLanes) o.src[s] = -1;
}

int bits_of(uint32_t most) {                         // bits that hold 0 .. most
  int b = 1;
  while (b < 32 && (most >> b) != 0) ++b;
  return b;
}
int64_t n_blocks(int64_t n) { return (n + kBlock - 1) / kBlock; }
constexpr int64_t kMostIds = 1ll << 20, kMostAssignments = 1ll << 22;

bool one_launch(int64_t n, int64_t V) { return n <= kMostAlone || (n <= kMostSplit && V <= kMostMarked); }

}  // namespace

extern "C" int64_t anc_id_groups_device_workspace_bytes(int64_t M, int64_t V) {
  if (M <= 0 || M > kMostIds || V <= 0 || V >= (1ll << 31)) {
    anc_set_error("anc_id_groups_device_workspace_bytes: M=%lld (1 .. %lld), V=%lld (1 .. 2^31 - 1)", (long long)M, (long long)kMostIds,
                  (long long)V);
    return -1;
  }
  if (one_launch(M, V)) return 16;
  const int64_t passes = (bits_of((uint32_t)V) + kDigitBits - 1) / kDigitBits;
  return 4 * (n_blocks(M) * (kDigits * passes + 1) + 4 * M);
}

extern "C" int anc_id_groups_device(uint64_t ids, int32_t ids_bytes, int64_t n, int64_t M, int64_t V, uint64_t srt, uint64_t start,
                             uint64_t cnt, uint64_t gid, uint64_t key, uint64_t grp, uint64_t count, uint64_t workspace,
                             int64_t workspace_bytes, uint64_t stream) {
  ANC_REQUIRE(M > 0 && M <= kMostIds && n >= 0 && n <= M && V > 0 && V < (1ll << 31),
              "anc_id_groups_device: n=%lld of M=%lld ids (at most %lld), V=%lld", (long long)n, (long long)M, (long long)kMostIds, (long long)V);
  ANC_REQUIRE(ids_bytes == 4 || ids_bytes == 8, "anc_id_groups_device: ids of %d bytes (4 or 8)", (int)ids_bytes);
  ANC_REQUIRE((ids != 0 || n == 0) && srt && start && cnt && gid && key && grp && count && workspace,
              "anc_id_groups_device: null pointer");
  ANC_REQUIRE(ids % (uint64_t)ids_bytes == 0 && ((srt | start | cnt | gid | key | grp | count) & 3) == 0 && (workspace & 15) == 0,
              "anc_id_groups_device: misaligned pointers");
  const int64_t ws = anc_id_groups_device_workspace_bytes(n > 0 ? n : 1, V);
  ANC_REQUIRE(workspace_bytes >= ws, "anc_id_groups_device: workspace holds %lld bytes, %lld needed", (long long)workspace_bytes, (long long)ws);
  // (workgroups read the ids more than once and write by what they found)
  ANC_REQUIRE(anc_outputs_apart({{srt, 4 * M}, {start, 4 * M}, {cnt, 4 * M}, {gid, 4 * M}, {key, 4 * M}, {grp, 4 * M}, {count, 4}, {workspace, ws},
                                 {ids, n * ids_bytes}}, 8),
              "anc_id_groups_device: an output or the workspace overlaps another buffer");
  hipStream_t s = anc_stream(stream);
  AncProfScope prof(ANC_PROF_MISC, s);
  const Groups o{(int32_t *)srt, (int32_t *)start, (int32_t *)cnt, (int32_t *)gid, (int32_t *)key, (int32_t *)grp, (int32_t *)count};
  const int bits = bits_of((uint32_t)V), wide = ids_bytes == 8;
  if (n <= kFewAlone) {
    if (wide) hipLaunchKernelGGL((k_group_part<256, false, int64_t>), dim3(1), dim3(256), 0, s, (const int64_t *)ids, (int)n, M, (uint32_t)V, o);
    else      hipLaunchKernelGGL((k_group_part<256, false, int32_t>), dim3(1), dim3(256), 0, s, (const int32_t *)ids, (int)n, M, (uint32_t)V, o);
    ANC_LAUNCH_CHECK();
    return ANC_OK;
  }
  if (n <= kMostAlone) {
    if (wide) hipLaunchKernelGGL((k_group_part<512, false, int64_t>), dim3(1), dim3(512), 0, s, (const int64_t *)ids, (int)n, M, (uint32_t)V, o);
    else      hipLaunchKernelGGL((k_group_part<512, false, int32_t>), dim3(1), dim3(512), 0, s, (const int32_t *)ids, (int)n, M, (uint32_t)V, o);
    ANC_LAUNCH_CHECK();
    return ANC_OK;
  }
  if (one_launch(n, V)) {
    const int64_t parts = (n + 31) / 32;
    const dim3 grid((unsigned)(parts < 128 ? parts : 128));
    const bool few = n <= kFewSplit;
    auto kernel = few ? k_group_part<512, true, int64_t> : k_group_part<1024, true, int64_t>;
    auto narrow = few ? k_group_part<512, true, int32_t> : k_group_part<1024, true, int32_t>;
    if (wide) hipLaunchKernelGGL(kernel, grid, dim3(few ? 512 : 1024), 0, s, (const int64_t *)ids, (int)n, M, (uint32_t)V, o);
    else      hipLaunchKernelGGL(narrow, grid, dim3(few ? 512 : 1024), 0, s, (const int32_t *)ids, (int)n, M, (uint32_t)V, o);
    ANC_LAUNCH_CHECK();
    return ANC_OK;
  }
  const int64_t blocks = n_blocks(n);
  const dim3 grid((unsigned)blocks), lanes(kBlockLanes);
  const int passes = (bits + kDigitBits - 1) / kDigitBits;
  int *hist = (int *)workspace, *heads = hist + blocks * kDigits * passes;
  int32_t *buf = heads + blocks;                     // two (key, position) pairs of arrays
  hipLaunchKernelGGL(k_radix_count, grid, lanes, 0, s, (const void *)ids, wide, n, M, (uint32_t)V, bits, passes, hist, o.cnt);
  const int32_t *key_in = nullptr, *idx_in = nullptr;
  for (int q = 0; q < passes; ++q) {
    const bool last = q + 1 == passes;
    int32_t *key_out = last ? o.key : buf + (q & 1) * 2 * n, *idx_out = last ? o.srt : key_out + n;
    hipLaunchKernelGGL(k_radix_scatter, grid, lanes, 0, s, (const void *)ids, wide, key_in, idx_in, n, (uint32_t)V,
                       q * kDigitBits, bits, (const int *)(hist + q * blocks * kDigits),
                       last ? (int *)nullptr : hist + (q + 1) * blocks * kDigits, key_out, idx_out);
    key_in = key_out;
    idx_in = idx_out;
  }
  hipLaunchKernelGGL(k_heads, grid, lanes, 0, s, (const int32_t *)o.key, n, (uint32_t)V, heads);
  hipLaunchKernelGGL(k_groups, grid, lanes, 0, s, n, M, (uint32_t)V, (const int *)heads, o);
  ANC_LAUNCH_CHECK();
  return ANC_OK;
}

static int check_route(const char *who, int64_t A, int64_t E, int64_t align, int64_t &capacity) {
  ANC_REQUIRE(A > 0 && A <= kMostAssignments && E > 0 && E <= kMostExperts && align > 0 && align <= 256 && (align & (align - 1)) == 0,
              "%s: %lld assignments (1 .. %lld) to %lld experts (1 .. %d), align %lld (a power of two up to 256)", who,
              (long long)A, (long long)kMostAssignments, (long long)E, kMostExperts, (long long)align);
  capacity = A + (E < A ? E : A) * (align - 1);
  return ANC_OK;
}

extern "C" int64_t anc_route_capacity(int64_t assignments, int64_t experts, int64_t align) {
  int64_t c;
  return check_route("anc_route_capacity", assignments, experts, align, c) ? -1 : c;
}

extern "C" int64_t anc_route_workspace_bytes(int64_t assignments, int64_t experts) {
  int64_t c;
  if (check_route("anc_route_workspace_bytes", assignments, experts, 1, c)) return -1;
  return assignments <= kMostCounted ? 4 : 4 * n_blocks(assignments) * experts;
}

extern "C" int anc_route(uint64_t expert_ids, int32_t ids_bytes, int64_t n, int64_t experts, int64_t align, uint64_t counts,
                         uint64_t offsets, uint64_t order, uint64_t slot, uint64_t src, int64_t capacity, uint64_t workspace,
                         int64_t workspace_bytes, uint64_t stream) {
  int64_t need;
  if (int rc = check_route("anc_route", n > 0 ? n : 1, experts, align, need)) return rc;
  ANC_REQUIRE(n >= 0 && capacity >= (n > 0 ? need : 1) && capacity < (1ll << 31), "anc_route: %lld assignments, room for %lld slots, %lld needed",
              (long long)n, (long long)capacity, (long long)need);
  ANC_REQUIRE(ids_bytes == 4 || ids_bytes == 8, "anc_route: ids of %d bytes (4 or 8)", (int)ids_bytes);
  ANC_REQUIRE((expert_ids != 0 || n == 0) && counts && offsets && order && slot && src && workspace, "anc_route: null pointer");
  ANC_REQUIRE(expert_ids % (uint64_t)ids_bytes == 0 && ((counts | offsets | order | slot | src | workspace) & 3) == 0,
              "anc_route: misaligned pointers");
  const int64_t ws = anc_route_workspace_bytes(n > 0 ? n : 1, experts);
  ANC_REQUIRE(workspace_bytes >= ws, "anc_route: workspace holds %lld bytes, %lld needed", (long long)workspace_bytes, (long long)ws);
  ANC_REQUIRE(anc_outputs_apart({{counts, 4 * experts}, {offsets, 4 * experts + 4}, {order, 4 * experts}, {slot, 4 * n}, {src, 4 * capacity},
                                 {workspace, ws}, {expert_ids, n * ids_bytes}}, 6),
              "anc_route: an output or the workspace overlaps another buffer");
  hipStream_t s = anc_stream(stream);
  AncProfScope prof(ANC_PROF_MISC, s);
  const Route o{(int32_t *)counts, (int32_t *)offsets, (int32_t *)order, (int32_t *)slot, (int32_t *)src};
  const int E = (int)experts, bits = bits_of((uint32_t)E - 1), wide = ids_bytes == 8;
  if (n <= kMostCounted) {
    hipLaunchKernelGGL(k_route_one, dim3((unsigned)(n > 0 ? (n + kOneLanes - 1) / kOneLanes : 1)), dim3(kOneLanes), 0, s, (const void *)expert_ids, wide, (int)n, E,
                       bits, (int)align, (int)capacity, o);
  } else {
    const dim3 grid((unsigned)n_blocks(n)), lanes(kBlockLanes);
    hipLaunchKernelGGL(k_route_count, grid, lanes, 0, s, (const void *)expert_ids, wide, n, E, (int *)workspace);
    hipLaunchKernelGGL(k_route_place, grid, lanes, 0, s, (const void *)expert_ids, wide, n, E, bits, (int)align, capacity,
                       (const int *)workspace, o);
  }
  ANC_LAUNCH_CHECK();
  return ANC_OK;
}
