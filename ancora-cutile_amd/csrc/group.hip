// Small integer keys put in order on the device: token ids into groups of one id, (token, choice) assignments into
// segments of one expert. Both are a stable sort, so that what is summed up over a group is summed in the tokens' order
// and the same on every run.
//
// Ranking: a wavefront takes 64 consecutive items at a time. The lanes that hold the same digit are found with one ballot
// per bit of the digit; an item's rank is the number of earlier lanes among them plus the wavefront's count of the digit
// so far, a counter in LDS. Items of different wavefronts meet in an exclusive sum over (digit, wavefront).
//
// Up to 1024 x kMostItems items one workgroup does everything in one launch: the keys stay in LDS and only 16-bit positions are
// permuted, 9 bits a pass (two passes for a vocabulary of 152 K). Beyond, the same passes run over blocks of kBlock items
// with the blocks' digit counts in memory: a block adds up the counts before it itself (no launch in between), and the
// count for the next pass is made by the scatter, with integer atomics, which have no order to lose.
#include "common.h"

namespace {

constexpr int kDigitBits = 9, kDigits = 1 << kDigitBits;
constexpr int kMostItems = 16;                       // per lane of the one-workgroup kernels
constexpr int kSmallMax = 1024 * kMostItems;
constexpr int kBlockLanes = 256, kBlockItems = 8, kBlock = kBlockLanes * kBlockItems;

// Lanes of the wavefront that hold the same digit as this one, among those with `in`. (Six vector instructions a bit: the digit's bit
// as 0 or -1, its ballot, and two words of agreement.)
__device__ __forceinline__ uint64_t same_digit(uint32_t d, int bits, bool in) {
  const uint64_t all = __ballot(in);
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
__device__ __forceinline__ int wave_scan(int v) {          // inclusive
  const int lane = (int)(threadIdx.x & 63);
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(v, o, 64);
    if (lane >= o) v += u;
  }
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

// ---------------------------------------------------------------- token ids, one workgroup
template <int ITEMS>
__global__ void __launch_bounds__(1024)
k_group_small(const void *__restrict__ ids, int wide, int n, int M, uint32_t V, int bits, Groups o) {
  constexpr int W = 16, N = 1024 * ITEMS;
  __shared__ uint32_t skey[N];
  __shared__ uint16_t sidx[N];
  __shared__ int count[W * kDigits];
  __shared__ int tmp[W];
  const int tid = (int)threadIdx.x, wave = tid >> 6, lane = tid & 63, first = wave * (64 * ITEMS) + lane;
  int idx[ITEMS];
  uint32_t key[ITEMS];
  if (n > 0) {
    load_keys<ITEMS>(ids, wide, first, 64, n, V, key);       // (what lies behind the last id stays behind the ids that name no row)
  } else {
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) key[j] = V;
  }
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    idx[j] = first + 64 * j;
    skey[first + 64 * j] = key[j];
  }
  for (int shift = 0; shift < bits; shift += kDigitBits) {
    const int b = bits - shift < kDigitBits ? bits - shift : kDigitBits, digits = 1 << b;
    for (int i = tid; i < W << b; i += 1024) count[i] = 0;
    __syncthreads();
    int rank[ITEMS];
#pragma unroll
    for (int j = 0; j < ITEMS; ++j)
      rank[j] = take_rank(count + (wave << b), (key[j] >> shift) & (digits - 1), b, true);
    __syncthreads();
    int c[W], sum = 0, total;
#pragma unroll
    for (int w = 0; w < W; ++w) c[w] = tid < digits ? count[(w << b) + tid] : 0;
#pragma unroll
    for (int w = 0; w < W; ++w) sum += c[w];
    int at = block_scan<1024>(sum, tmp, total);
    if (tid < digits) {
#pragma unroll
      for (int w = 0; w < W; ++w) {
        count[(w << b) + tid] = at;
        at += c[w];
      }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < ITEMS; ++j)
      sidx[count[(wave << b) + ((key[j] >> shift) & (digits - 1))] + rank[j]] = (uint16_t)idx[j];
    __syncthreads();
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
      idx[j] = sidx[first + 64 * j];
      key[j] = skey[idx[j]];
    }
  }
  // The number of heads (first items of an id) up to an item is its group.
  int heads = 0, valid = 0, mine = 0;
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    const int p = first + 64 * j;
    const bool head = key[j] < V && (p == 0 || skey[sidx[p - 1]] != key[j]);
    heads |= head ? 1 << j : 0;
    mine += head ? 1 : 0;
    valid += key[j] < V ? 1 : 0;
  }
  int total, n_valid;
  const int before = block_scan<1024>(mine, tmp, total) - (wave_scan(mine) - mine);    // heads of the wavefronts before this one
  block_scan<1024>(valid, tmp, n_valid);             // (its barriers also end the reads of skey above)
  int run = before;
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    const int p = first + 64 * j;
    const bool head = (heads >> j) & 1;
    const uint64_t m = __ballot(head);
    const int g = run + __popcll(m & ((1ull << lane) - 1)) - (head ? 0 : 1);
    run += __popcll(m);
    if (p < n) {
      o.srt[p] = idx[j];
      o.key[p] = (int32_t)key[j];
      o.grp[p] = key[j] < V ? g : -1;
    }
    if (head) {
      skey[g] = (uint32_t)p;
      o.gid[g] = (int32_t)key[j];
    }
  }
  __syncthreads();
  for (int g = tid; g < M; g += 1024) {
    const bool used = g < total;
    const int at = used ? (int)skey[g] : 0;
    o.start[g] = at;
    o.cnt[g] = used ? (g + 1 < total ? (int)skey[g + 1] : n_valid) - at : 0;
    if (!used) o.gid[g] = -1;
  }
  if (tid == 0) *o.count = total;
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

// Items [lo, lo + 64 * ITEMS) of a wavefront in rank order; `base`: first place of every digit for this block.
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
#pragma unroll 8
  for (int64_t c = 0; c < blocks; ++c) {
#pragma unroll
    for (int q = 0; q < PER; ++q) {
      const int v = hist[c * kDigits + tid * PER + q];
      all[q] += v;
      below[q] += c < b ? v : 0;
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
// by looking at all of them (LANES / E lanes share the looking). Beyond kMostOrdered that would take longer than it gives: many
// short segments even out in any order.
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
  for (int j = (int)threadIdx.x % L; j < E; j += L) {
    const int c = scnt[j];
    before += c > mine || (c == mine && j < e) ? 1 : 0;
  }
#pragma unroll
  for (int o = 1; o < L; o <<= 1) before += __shfl_xor(before, o, 64);
  if (e < E && (int)threadIdx.x % L == 0) order[before] = e;
}
__device__ __forceinline__ int filled_up(int c, int align) { return (c + align - 1) & -align; }

template <int ITEMS>
__global__ void __launch_bounds__(1024)
k_route_small(const void *__restrict__ ids, int wide, int n, int E, int bits, int align, int capacity, Route o) {
  constexpr int W = 16;
  __shared__ int count[W * kMostExperts];
  __shared__ int tmp[W];
  __shared__ int soff[kMostExperts + 1], scnt[kMostExperts];
  const int tid = (int)threadIdx.x, wave = tid >> 6, lane = tid & 63, first = wave * (64 * ITEMS) + lane;
  uint32_t e[ITEMS];                                 // E: no expert
  int rank[ITEMS];
  if (n > 0) {
    load_keys<ITEMS>(ids, wide, first, 64, n, (uint32_t)E, e);
  } else {
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) e[j] = (uint32_t)E;
  }
  for (int i = tid; i < W * E; i += 1024) count[i] = 0;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) rank[j] = take_rank(count + wave * E, e[j], bits, e[j] < (uint32_t)E);
  __syncthreads();
  int c[W], sum = 0, total;
#pragma unroll
  for (int w = 0; w < W; ++w) c[w] = tid < E ? count[w * E + tid] : 0;
#pragma unroll
  for (int w = 0; w < W; ++w) sum += c[w];
  const int base = block_scan<1024>(filled_up(sum, align), tmp, total);
  if (tid < E) {
    int at = base;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      count[w * E + tid] = at;
      at += c[w];
    }
    soff[tid] = base;
    scnt[tid] = sum;
    o.counts[tid] = sum;
    o.offsets[tid] = base;
  }
  if (tid == 0) { soff[E] = total; o.offsets[E] = total; }
  __syncthreads();
  order_experts<1024>(scnt, E, o.order);
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    const int p = first + 64 * j;
    if (p >= n) continue;
    const int s = e[j] < (uint32_t)E ? count[wave * E + e[j]] + rank[j] : -1;
    o.slot[p] = s;
    if (s >= 0) o.src[s] = p;
  }
  for (int q = wave; q < E; q += W)
    for (int s = soff[q] + scnt[q] + lane; s < soff[q + 1]; s += 64) o.src[s] = -1;
  for (int s = total + tid; s < capacity; s += 1024) o.src[s] = -1;
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
  __shared__ int soff[kMostExperts + 1], scnt[kMostExperts];
  const int tid = (int)threadIdx.x, wave = tid >> 6, lane = tid & 63, blocks = (int)gridDim.x, b = (int)blockIdx.x;
  const int64_t first = (int64_t)b * kBlock + wave * (64 * kBlockItems) + lane;
  uint32_t e[kBlockItems];
  int rank[kBlockItems], all[PER], below[PER];
  load_keys<kBlockItems>(ids, wide, first, 64, n, (uint32_t)E, e);
  for (int i = tid; i < W * E; i += kBlockLanes) count[i] = 0;
#pragma unroll
  for (int q = 0; q < PER; ++q) {
    all[q] = below[q] = 0;
    const int d = tid * PER + q;
    if (d < E) {
#pragma unroll 8
      for (int c = 0; c < blocks; ++c) {
        const int v = hist[(int64_t)c * E + d];
        all[q] += v;
        below[q] += c < b ? v : 0;
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kBlockItems; ++j)
    rank[j] = take_rank(count + wave * E, e[j], bits, e[j] < (uint32_t)E);
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

template <int V> struct IC { static constexpr int value = V; };
template <typename F> void with_items(int64_t n, F &&f) {
  if (n <= 1024) f(IC<1>{}); else if (n <= 4096) f(IC<4>{}); else if (n <= 8192) f(IC<8>{}); else f(IC<kMostItems>{});
}

}  // namespace

extern "C" int64_t anc_id_groups_device_workspace_bytes(int64_t M, int64_t V) {
  if (M <= 0 || M > kMostIds || V <= 0 || V >= (1ll << 31)) {
    anc_set_error("anc_id_groups_device_workspace_bytes: M=%lld (1 .. %lld), V=%lld (1 .. 2^31 - 1)", (long long)M, (long long)kMostIds,
                  (long long)V);
    return -1;
  }
  const int64_t passes = (bits_of((uint32_t)V) + kDigitBits - 1) / kDigitBits;
  return M <= kSmallMax ? 4 : 4 * (n_blocks(M) * (kDigits * passes + 1) + 4 * M);
}

extern "C" int anc_id_groups_device(uint64_t ids, int32_t ids_bytes, int64_t n, int64_t M, int64_t V, uint64_t srt, uint64_t start,
                             uint64_t cnt, uint64_t gid, uint64_t key, uint64_t grp, uint64_t count, uint64_t workspace,
                             int64_t workspace_bytes, uint64_t stream) {
  ANC_REQUIRE(M > 0 && M <= kMostIds && n >= 0 && n <= M && V > 0 && V < (1ll << 31),
              "anc_id_groups_device: n=%lld of M=%lld ids (at most %lld), V=%lld", (long long)n, (long long)M, (long long)kMostIds, (long long)V);
  ANC_REQUIRE(ids_bytes == 4 || ids_bytes == 8, "anc_id_groups_device: ids of %d bytes (4 or 8)", (int)ids_bytes);
  ANC_REQUIRE((ids != 0 || n == 0) && srt && start && cnt && gid && key && grp && count && workspace,
              "anc_id_groups_device: null pointer");
  ANC_REQUIRE(ids % (uint64_t)ids_bytes == 0 && ((srt | start | cnt | gid | key | grp | count | workspace) & 3) == 0,
              "anc_id_groups_device: misaligned pointers");
  ANC_REQUIRE(workspace_bytes >= anc_id_groups_device_workspace_bytes(n > 0 ? n : 1, V), "anc_id_groups_device: workspace holds %lld bytes, %lld needed",
              (long long)workspace_bytes, (long long)anc_id_groups_device_workspace_bytes(n > 0 ? n : 1, V));
  hipStream_t s = anc_stream(stream);
  AncProfScope prof(ANC_PROF_MISC, s);
  const Groups o{(int32_t *)srt, (int32_t *)start, (int32_t *)cnt, (int32_t *)gid, (int32_t *)key, (int32_t *)grp, (int32_t *)count};
  const int bits = bits_of((uint32_t)V), wide = ids_bytes == 8;
  if (n <= kSmallMax) {
    with_items(n, [&](auto items) {
      hipLaunchKernelGGL(k_group_small<decltype(items)::value>, dim3(1), dim3(1024), 0, s, (const void *)ids, wide, (int)n, (int)M,
                         (uint32_t)V, bits, o);
    });
    ANC_LAUNCH_CHECK();
    return ANC_OK;
  }
  const int64_t blocks = n_blocks(n);
  const int passes = (bits + kDigitBits - 1) / kDigitBits;
  int *hist = (int *)workspace, *heads = hist + blocks * kDigits * passes;
  int32_t *buf = heads + blocks;                     // two (key, position) pairs of arrays
  const dim3 grid((unsigned)blocks), lanes(kBlockLanes);
  hipLaunchKernelGGL(k_radix_count, grid, lanes, 0, s, (const void *)ids, wide, n, M, (uint32_t)V, bits, passes, hist, o.cnt);
  const int32_t *key_in = nullptr, *idx_in = nullptr;
  for (int q = 0; q < passes; ++q) {
    const bool last = q + 1 == passes;
    int32_t *key_out = last ? o.key : buf + (q & 1) * 2 * n, *idx_out = last ? o.srt : key_out + n;
    hipLaunchKernelGGL(k_radix_scatter, grid, lanes, 0, s, (const void *)ids, wide, key_in, idx_in, n, (uint32_t)V,
                       q * kDigitBits, bits, hist + q * blocks * kDigits, last ? (int *)nullptr : hist + (q + 1) * blocks * kDigits,
                       key_out, idx_out);
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
  return assignments <= kSmallMax ? 4 : 4 * n_blocks(assignments) * experts;
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
  hipStream_t s = anc_stream(stream);
  AncProfScope prof(ANC_PROF_MISC, s);
  const Route o{(int32_t *)counts, (int32_t *)offsets, (int32_t *)order, (int32_t *)slot, (int32_t *)src};
  const int E = (int)experts, bits = bits_of((uint32_t)E - 1), wide = ids_bytes == 8;
  if (n <= kSmallMax) {
    with_items(n, [&](auto items) {
      hipLaunchKernelGGL(k_route_small<decltype(items)::value>, dim3(1), dim3(1024), 0, s, (const void *)expert_ids, wide, (int)n, E,
                         bits, (int)align, (int)capacity, o);
    });
  } else {
    const dim3 grid((unsigned)n_blocks(n)), lanes(kBlockLanes);
    hipLaunchKernelGGL(k_route_count, grid, lanes, 0, s, (const void *)expert_ids, wide, n, E, (int *)workspace);
    hipLaunchKernelGGL(k_route_place, grid, lanes, 0, s, (const void *)expert_ids, wide, n, E, bits, (int)align, capacity,
                       (const int *)workspace, o);
  }
  ANC_LAUNCH_CHECK();
  return ANC_OK;
}
