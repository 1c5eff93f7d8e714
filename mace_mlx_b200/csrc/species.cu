// Species operators that move rows: stable grouping by species, the node
// embedding and its table gradient, and the 8-bit row checkpoint
// (species_linear.cu holds the species-indexed linear map).
//
// What they restate (paths in the reference project):
//   node embedding (one-hot linear)  mace_mlx/model.py:373-438
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "common.cuh"
#include "species.cuh"

namespace mace {

namespace {

// row movers: threads of a CTA and vectors per thread (loads in flight)
constexpr int RW_THREADS = 256;
constexpr int RW_UNROLL = 4;
constexpr int RS_UNROLL = 4;  // of the restore

// x / C for x < 2^32 / C by multiplication: the row of a CTA's local element
// (x < RW_THREADS RW_UNROLL 8 + C and C <= 32768 stay below the limit)
struct RowDiv {
  uint32_t mul, one;
  __device__ __forceinline__ uint32_t quotient(uint32_t x) const { return one ? x : __umulhi(x, mul); }
};
RowDiv row_div(int C) { return {(uint32_t)((((uint64_t)1 << 32) + C - 1) / C), C == 1 ? 1u : 0u}; }

// Grouping is a stable counting sort by the key (species, or num_groups for
// padding rows): one pass for keys of up to 13 bits, else two passes over half
// the bits each.  A pass counts the digits of every CTA's share of the list,
// scans the counts over the CTAs, and scatters: a warp takes consecutive rows,
// ranks them among equal digits with ballots and moves its own counter of the
// digit on (16 bits in shared memory: a share has fewer rows).  Ranks follow
// the list order everywhere, so the order of atomics plays no part.
//
// 4M rows, 7921 groups: 45 us, of which the scatter is two thirds, bound by its
// 4-byte stores (a sector each) and the latency of its few warps; in two
// passes of 7 bits, put in digit order in shared memory before they are
// stored, 98 us.  1000 groups: 38 us (89 in two passes); 89 groups: 36 us (40).
// 16 000 groups take two passes (101 us): the counters of 14 bits would leave
// shared memory for 5 warps.
constexpr int GR_THREADS = 1024;  // of the counting and scanning CTAs
constexpr int GR_MAX_BITS = 13;   // digit of one pass: the counters of 12 warps fill the shared memory
constexpr int GR_CTAS = 148;      // one per SM
template <int BITS>
struct GroupCfg {
  static constexpr int BINS = 1 << BITS, WORDS = BINS / 2;
  static constexpr int WARPS = BITS == 13 ? 12 : (BITS == 12 ? 24 : 32), THREADS = WARPS * 32;
  static constexpr int BYTES = (BINS + WARPS * WORDS + 32) * 4;
  static_assert(BYTES <= 232448, "shared memory of a CTA");
};
// short lists: one CTA does the whole sort in one launch (89 groups: 1000 rows 3.5 us against 6.3 in three launches,
// 4096 rows 6.2 against 7.9, 8192 rows 10.1 against 8.3)
constexpr int GS_THREADS = 1024;
constexpr int GS_MAX_ROWS = 6144;
constexpr int GS_MAX_BINS = 256;  // (shared memory of a static size)

// key of a row: its species, or num_groups for padding rows
__device__ __forceinline__ int row_key(int32_t z, int G) { return (z >= 0 && z < G) ? z : G; }

struct GroupPass {
  const int32_t* species;
  const int2* in;       // second pass: (key, row) sorted by the lower digit; null in the first: row i is i
  int64_t n;
  int G;
  int shift, bits;
  int share, nb;        // rows of a CTA (a multiple of its threads, below 2^16), CTAs
  int32_t* counts;      // (nb, bins), after the scan exclusive within a digit
  int32_t* totals;      // (bins)
  int2* out;            // first pass of two: (key, row), one scattered store; else null
  int32_t* order;
  int32_t* offsets;     // single pass: the group offsets; else null
};

__device__ __forceinline__ int key_of(const GroupPass& p, int64_t i) {
  return p.in ? p.in[i].x : row_key(p.species[i], p.G);
}
__device__ __forceinline__ int digit_of(const GroupPass& p, int key) { return (key >> p.shift) & ((1 << p.bits) - 1); }

__global__ void __launch_bounds__(GR_THREADS) k_group_count(GroupPass p) {
  __shared__ int hist[1 << GR_MAX_BITS];
  const int bins = 1 << p.bits;
  for (int b = threadIdx.x; b < bins; b += GR_THREADS) hist[b] = 0;
  pdl_wait();
  __syncthreads();
  const int64_t i0 = blockIdx.x * (int64_t)p.share;
  const int rows = (int)imin64(p.share, p.n - i0);
#pragma unroll 8
  for (int i = threadIdx.x; i < rows; i += GR_THREADS) atomicAdd(&hist[digit_of(p, key_of(p, i0 + i))], 1);
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += GR_THREADS) p.counts[(int64_t)blockIdx.x * bins + b] = hist[b];
}

// exclusive sums of the counts of 32 digits over the CTAs, in place, and their totals: a lane per digit, each warp a
// run of CTAs
__global__ void __launch_bounds__(GR_THREADS) k_group_scan(GroupPass p) {
  pdl_wait();
  __shared__ int sums[32][33];
  const int bins = 1 << p.bits, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int b = blockIdx.x * 32 + lane;
  const int per = (p.nb + 31) / 32, c0 = warp * per, c1 = min(p.nb, c0 + per);
  int32_t* const c = p.counts + b;
  int sum = 0;
  if (b < bins)
#pragma unroll 8
    for (int k = c0; k < c1; ++k) sum += c[(int64_t)k * bins];
  sums[warp][lane] = sum;
  __syncthreads();
  int at = 0;
  for (int w = 0; w < warp; ++w) at += sums[w][lane];
  if (b >= bins) return;
  if (warp == 31) p.totals[b] = at + sum;
#pragma unroll 8
  for (int k = c0; k < c1; ++k) {
    const int v = c[(int64_t)k * bins];
    c[(int64_t)k * bins] = at;
    at += v;
  }
}

// exclusive sums over `count` values of a CTA's threads, thread by thread: value v, result returned
template <int THREADS>
__device__ __forceinline__ int cta_exclusive(int v, int* warp_sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += u;
  }
  if (lane == 31) warp_sums[warp] = s;
  __syncthreads();
  int before = 0;
  for (int w = 0; w < warp; ++w) before += warp_sums[w];
  __syncthreads();
  return before + s - v;
}

// The lanes (of those with `in`) whose digit is this lane's.  They find one another bit by bit with ballots (match_any
// on spread digits costs several times as much).
template <int BITS>
__device__ __forceinline__ unsigned same_digit(int digit, bool in) {
  unsigned same = __ballot_sync(0xffffffffu, in);
#pragma unroll
  for (int b = 0; b < BITS; ++b) {
    const bool one = (digit >> b) & 1;
    const unsigned m = __ballot_sync(0xffffffffu, one);
    same &= one ? m : ~m;
  }
  return same;
}

// Place of this lane's row among its warp's rows of the same digit: `count` holds how many came before, and is moved
// on.
template <typename C>
__device__ __forceinline__ int place(C* count, int digit, bool in, unsigned same, int lane) {
  const int rank = __popc(same & ((1u << lane) - 1));
  const int before = in ? count[digit] : 0;
  __syncwarp();
  if (in && rank == 0) count[digit] = (C)(before + __popc(same));
  __syncwarp();
  return before + rank;
}

template <int BITS>
__global__ void __launch_bounds__(GroupCfg<BITS>::THREADS, 1) k_group_scatter(GroupPass p) {
  using Cfg = GroupCfg<BITS>;
  constexpr int BINS = Cfg::BINS, WORDS = Cfg::WORDS, WARPS = Cfg::WARPS, THREADS = Cfg::THREADS;
  extern __shared__ int32_t dyn[];
  int* const base = dyn;                                           // a digit's first position of this CTA
  uint32_t* const pos = reinterpret_cast<uint32_t*>(dyn + BINS);   // (WARPS, BINS) of 16 bits: counts, then positions
  int* const sums = dyn + BINS + WARPS * WORDS;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  for (int k = tid; k < WARPS * WORDS; k += THREADS) pos[k] = 0;
  pdl_wait();
  constexpr int PER = (BINS + THREADS - 1) / THREADS;
  int before[PER];  // this CTA's counts of digits tid + k THREADS
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int b = tid + k * THREADS;
    if (b < BINS) base[b] = p.totals[b];
    before[k] = b < BINS ? p.counts[(int64_t)blockIdx.x * BINS + b] : 0;
  }
  __syncthreads();
  const int seg = p.share / WARPS;  // consecutive rows of one warp
  const int64_t i0 = blockIdx.x * (int64_t)p.share + warp * seg;
  const int rows = (int)max(imin64(seg, p.n - i0), (int64_t)0);
  uint32_t* const mine = pos + warp * WORDS;
#pragma unroll 8
  for (int i = lane; i < rows; i += 32) {
    const int d = digit_of(p, key_of(p, i0 + i));
    atomicAdd(&mine[d >> 1], 1u << (16 * (d & 1)));
  }
  // exclusive sums over the digits, PER neighbours per thread
  int sum = 0;
#pragma unroll
  for (int k = 0; k < PER; ++k) sum += tid * PER + k < BINS ? base[tid * PER + k] : 0;
  sum = cta_exclusive<THREADS>(sum, sums);
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int b = tid * PER + k;
    if (b >= BINS) break;
    const int total = base[b];
    base[b] = sum;
    sum += total;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int b = tid + k * THREADS;
    if (b >= BINS) break;
    const int at = base[b];
    if (p.offsets && blockIdx.x == 0 && b <= p.G) p.offsets[b] = at;
    base[b] = at + before[k];
  }
  // (cta_exclusive's barriers stand between the counts and this)
  for (int k = tid; k < WORDS; k += THREADS) {  // two digits at a time: neither half overflows
    uint32_t at = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const uint32_t c = pos[w * WORDS + k];
      pos[w * WORDS + k] = at;
      at += c;
    }
  }
  __syncthreads();
  constexpr int U = 4;  // rounds of 32 rows in flight
  // (4M rows of 4000 groups 40 us, 49 by ballots; of 1000 no difference)
  constexpr bool SPREAD = BITS >= 12;
  int z[U], r[U];
  auto load = [&](int i) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = i + u * 32 + lane;
      int2 v = make_int2(0, (int)(i0 + k));
      if (k < rows) {
        if (p.in)
          v = p.in[i0 + k];
        else
          v.x = p.species[i0 + k];  // (its key is taken when it is used: nothing waits for the load here)
      }
      z[u] = v.x, r[u] = v.y;
    }
  };
  load(0);
#pragma unroll 1
  for (int i = 0; i < rows; i += U * 32) {
    int k0[U], r0[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      k0[u] = p.in ? z[u] : row_key(z[u], p.G);
      r0[u] = r[u];
    }
    load(i + U * 32);
    // The counters of U rounds in order, none waiting for the one before.  Spread digits: every row counts itself, and
    // where two met (a counter is further on than its own addition) the lanes of equal digit are found afterwards;
    // else they are found first and one of them counts them all.
    unsigned same[U];
    uint32_t first[U], last[U];  // rows of the digit before this one (before its lanes); SPREAD: after the round
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool in = i + u * 32 + lane < rows;
      const int d = digit_of(p, k0[u]), half = 16 * (d & 1);
      volatile uint32_t* const word = mine + (d >> 1);
      first[u] = last[u] = 0;
      if constexpr (SPREAD) {
        if (in) first[u] = atomicAdd(const_cast<uint32_t*>(word), 1u << half) >> half & 0xffffu;
        __syncwarp();
        if (in) last[u] = *word >> half & 0xffffu;
        __syncwarp();
      } else {
        same[u] = same_digit<BITS>(d, in);
        if (in) first[u] = *word >> half & 0xffffu;
        __syncwarp();
        if (in && (same[u] & ((1u << lane) - 1)) == 0)
          atomicAdd(const_cast<uint32_t*>(word), (uint32_t)__popc(same[u]) << half);
        __syncwarp();
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool in = i + u * 32 + lane < rows;
      const int d = digit_of(p, k0[u]);
      int at = base[d] + (int)first[u];
      if constexpr (SPREAD) {
        if (__any_sync(0xffffffffu, in && last[u] != first[u] + 1)) {
          same[u] = same_digit<BITS>(d, in);
          at = base[d] + (int)last[u] - __popc(same[u]) + __popc(same[u] & ((1u << lane) - 1));
        }
      } else {
        at += __popc(same[u] & ((1u << lane) - 1));
      }
      if (in) {
        if (p.out)
          p.out[at] = make_int2(k0[u], r0[u]);
        else
          p.order[at] = r0[u];
      }
    }
  }
}

template <int BITS>
__global__ void __launch_bounds__(GS_THREADS) k_group_small(const int32_t* species, int n, int G, int32_t* order,
                                                            int32_t* offsets) {
  pdl_wait();
  __shared__ int whist[32][1 << BITS];
  __shared__ int sums[32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  constexpr int MOST = GS_MAX_ROWS / GS_THREADS;  // rounds of 32 rows of one warp
  const int rounds = (n + GS_THREADS - 1) / GS_THREADS;
  const int i0 = warp * rounds * 32, i1 = min(n, i0 + rounds * 32);  // consecutive rows of one warp
  int key[MOST], rel[MOST];
#pragma unroll
  for (int j = 0; j < MOST; ++j) key[j] = i0 + j * 32 + lane < i1 ? row_key(load_in(species + i0 + j * 32 + lane), G) : 0;
  for (int b = lane; b < (1 << BITS); b += 32) whist[warp][b] = 0;
  __syncwarp();
#pragma unroll
  for (int j = 0; j < MOST; ++j)
    if (j < rounds) {
      const bool in = i0 + j * 32 + lane < i1;
      rel[j] = place(whist[warp], key[j], in, same_digit<BITS>(key[j], in), lane);
    }
  __syncthreads();
  int total = 0;
  if (tid < (1 << BITS))
#pragma unroll 8
    for (int w = 0; w < 32; ++w) total += whist[w][tid];
  int at = cta_exclusive<GS_THREADS>(total, sums);
  if (tid < (1 << BITS)) {
    if (tid <= G) offsets[tid] = at;
#pragma unroll 8
    for (int w = 0; w < 32; ++w) {
      const int c = whist[w][tid];
      whist[w][tid] = at;
      at += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < MOST; ++j) {
    const int i = i0 + j * 32 + lane;
    if (j < rounds && i < i1) order[whist[warp][key[j]] + rel[j]] = i;
  }
}

// Two passes: offsets[v] = first position of the order whose key is >= v, a thread per offset (a pass over the keys
// that writes an offset where the key changes leaves one thread all the writes of a long run of empty groups: 4M rows
// that use 3 of 1M groups 3685 us, 115 so)
__global__ void __launch_bounds__(256) k_group_offsets(const int32_t* species, const int32_t* order, int64_t n, int G,
                                                       int32_t* offsets) {
  pdl_wait();
  const int v = blockIdx.x * 256 + threadIdx.x;
  if (v > G) return;
  int64_t lo = 0, hi = n;
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (row_key(load_in(species + load_in(order + mid)), G) < v)
      lo = mid + 1;
    else
      hi = mid;
  }
  offsets[v] = (int32_t)lo;
}

// out[i] = scale table[species[i]].  The table stays in L2 and the result's stores are the bound: 1M rows of 128 fp32
// channels 77 us, 6.7 TB/s (90 with 5 or 6 CTAs of 256 threads on an SM instead of 7); of 128 bf16 channels 45.
// Consecutive vectors of V elements of the (n, C) result, CTA by CTA.
// FLAT = 0: C is a multiple of V and every row is vector-aligned, so a vector
// lies in one row; FLAT = 1: the result is contiguous and a vector may pass a
// row's end (any C); V = 1 serves everything else.  ODD: the scale is not finite, and padding is zero all the same (its
// own variant: the choice per vector costs 2 of 45 us in bf16).
template <typename T, int V, bool FLAT, bool ODD = false>
__global__ void __launch_bounds__(RW_THREADS, V == 8 && FLAT ? 5 : 7)
    k_embed(const T* table, int64_t ts, int G, int C, const int32_t* species, int64_t n, float scale, T* out, int64_t os,
            RowDiv div) {
  pdl_wait();
  const int64_t v0 = blockIdx.x * (int64_t)(RW_THREADS * RW_UNROLL);  // first vector of this CTA
  const int64_t total = n * C;
  const int64_t row0 = (v0 * V) / C;
  const uint32_t first = (uint32_t)(v0 * V - row0 * C);
  uint32_t row[RW_UNROLL], col[RW_UNROLL];
  int z[RW_UNROLL];
  Raw<T, V> x[RW_UNROLL];  // !FLAT: as loaded
  float v[FLAT ? RW_UNROLL : 1][FLAT ? V : 1];
#pragma unroll
  for (int j = 0; j < RW_UNROLL; ++j) {
    const uint32_t local = first + (threadIdx.x + j * RW_THREADS) * V;
    row[j] = div.quotient(local), col[j] = local - row[j] * C;
    z[j] = v0 * V + (threadIdx.x + j * RW_THREADS) * V < total ? load_in(species + row0 + row[j]) : -1;
  }
#pragma unroll
  for (int j = 0; j < RW_UNROLL; ++j) {
    const int64_t at = v0 * V + (threadIdx.x + j * RW_THREADS) * V;
    if constexpr (!FLAT) {
      if (z[j] >= 0 && z[j] < G)
        x[j].load(table + z[j] * ts + col[j]);
      else
        x[j].zero();
    } else if (at < total) {
      uint32_t r = row[j], c = col[j];
      int t = z[j];
#pragma unroll
      for (int k = 0; k < V; ++k) {
        v[j][k] = t >= 0 && t < G ? scale * to_f32(load_in(table + t * ts + c)) : 0.f;
        if (++c == (uint32_t)C) {
          c = 0;
          ++r;
          t = row0 + r < n ? load_in(species + row0 + r) : -1;
        }
      }
    }
  }
#pragma unroll
  for (int j = 0; j < RW_UNROLL; ++j) {
    const int64_t at = v0 * V + (threadIdx.x + j * RW_THREADS) * V;
    if (at >= total) continue;
    if constexpr (!FLAT) {
      float u[V];
      x[j].values(u);
      const float by = !ODD || (z[j] >= 0 && z[j] < G) ? scale : 0.f;
#pragma unroll
      for (int k = 0; k < V; ++k) u[k] *= by;
      store_channels<T, V>(out + (row0 + row[j]) * os + col[j], u);
    } else {
      if (at + V <= total)
        store_channels<T, V>(out + at, v[j]);
      else
#pragma unroll
        for (int k = 0; k < V; ++k)
          if (at + k < total) out[at + k] = from_f32<T>(v[j][k]);
    }
  }
}

// Table gradient: each warp sums a contiguous share of the grouped rows, group
// by group, so a group inside one share is final; the first and the last group
// of a share may continue in its neighbours and go to two partial rows per
// warp, which k_embed_grad_join adds in share order.  Lanes hold V channels
// each; with few channels RL row lanes of a warp take every RL-th row and are
// joined by shuffles at a group's end.
struct EmbedGrad {
  const void* dy;
  int64_t ds;
  const int32_t* order;
  const int32_t* offsets;
  int64_t n;
  int G, C;
  int64_t share;   // rows of one warp
  int64_t shares;  // warps
  float scale;
  void* out;       // (G, C)
  float* part;     // (shares, 2, C)
};

// group of grouped position i: the largest g with offsets[g] <= i (G: past the last group); by a whole warp, 32 places
// at a time
__device__ __forceinline__ int group_at(const int32_t* offsets, int G, int64_t i) {
  const int lane = threadIdx.x & 31;
  int lo = 0, count = G + 1;  // the group is one of lo .. lo + count - 1
  while (count > 1) {
    const int step = (count + 31) / 32;
    const int at = lo + lane * step;
    const unsigned below = __ballot_sync(0xffffffffu, lane == 0 || (lane * step < count && offsets[at] <= i));
    const int last = 31 - __clz(below);
    count = min(step, count - last * step);
    lo += last * step;
  }
  return lo;
}

constexpr int EG_THREADS = 256;

// A warp sums its share of the grouped list, V channels per lane and RL rows side by side.  The list is read and its
// rows are loaded UN RL at a time whatever groups they belong to; a group's end only cuts the additions, so that no
// load waits for a group before it.  1M fp32 rows of 128 channels: 4 groups 86 us with the join, 7921 groups 103 (79 is
// what HBM needs; group by group 92 and 112).  APART: rows that are not whole 16-byte pieces, a lane's channels 32
// apart, so that a warp still has 128 channels of 8 rows in flight: 1M rows of 97 channels fp32 87 us, bf16 78 (with
// one channel per lane 212 and 178).  A lane sums 32 rows of the list and then those sums: in one sum of its share the
// error at 1e8 rows of 17 channels was past 2.6e-6 of the result (3e-7 so, at no cost).
template <typename T, int V, int RL, bool APART = false>
__global__ void __launch_bounds__(EG_THREADS, 3) k_embed_grad(EmbedGrad p) {
  pdl_wait();
  constexpr int CL = 32 / RL;          // channel lanes
  constexpr int UN = RL == 8 ? 4 : 8;  // row loads in flight per lane
  constexpr int HOP = APART ? CL : 1;  // from one channel of a lane to the next
  constexpr int R = UN * RL;           // rows at a time (at most 32)
  const int lane = threadIdx.x & 31, cl = lane % CL, rl = lane / CL;
  const int64_t share = blockIdx.x * (int64_t)(EG_THREADS / 32) + (threadIdx.x >> 5);
  if (share >= p.shares) return;
  const int c0 = APART ? blockIdx.y * CL * V + cl : (blockIdx.y * CL + cl) * V;
  const bool in = c0 < p.C;
  // (positions in 32 bits: n < 2^31, and none passes n by more than 64)
  const uint32_t i0 = (uint32_t)(share * p.share), i1 = (uint32_t)imin64(p.n, share * p.share + p.share);
  const uint32_t stop = min(i1, (uint32_t)max(p.offsets[p.G], 0));  // padding rows are last
  if (i0 >= stop) return;
  const T* dy = static_cast<const T*>(p.dy) + (in ? c0 : 0);
  int32_t next = i0 + lane < stop ? p.order[i0 + lane] : -1;
  int g = group_at(p.offsets, p.G, i0);
  // offsets of 32 groups from `base` on
  int base = g;
  int32_t window = p.offsets[min(base + lane, p.G)];
  auto offset = [&](int k) -> uint32_t {  // k >= base
    if (k - base > 31) {
      base = k - 1;
      window = p.offsets[min(base + lane, p.G)];
    }
    return max(__shfl_sync(0xffffffffu, window, k - base), 0);
  };
  uint32_t lo = offset(g), hi = offset(g + 1);
  bool first = true;
  float acc[V] = {}, sum[V] = {};  // of the last 32 rows (at most), of those before them
  auto flush = [&]() {
#pragma unroll
    for (int k = 0; k < V; ++k) acc[k] += sum[k];
#pragma unroll
    for (int o = CL; o < 32; o <<= 1)
#pragma unroll
      for (int k = 0; k < V; ++k) acc[k] += __shfl_xor_sync(0xffffffffu, acc[k], o);
    if (rl == 0 && in) {
      if (lo >= i0 && hi <= i1) {
#pragma unroll
        for (int k = 0; k < V; ++k) acc[k] *= p.scale;
        T* const out = static_cast<T*>(p.out) + (int64_t)g * p.C + c0;
        if constexpr (APART) {
#pragma unroll
          for (int k = 0; k < V; ++k)
            if (k * HOP < p.C - c0) out[k * HOP] = from_f32<T>(acc[k]);
        } else {
          store_channels<T, V>(out, acc);
        }
      } else {
        float* part = p.part + (share * 2 + (first ? 0 : 1)) * p.C + c0;
#pragma unroll
        for (int k = 0; k < V; ++k)
          if (!APART || k * HOP < p.C - c0) part[k * HOP] = acc[k];
      }
    }
#pragma unroll
    for (int k = 0; k < V; ++k) acc[k] = sum[k] = 0.f;
    first = false;
  };
  Raw<T, V, APART> v[UN];
  int32_t mine = 0;
  auto load = [&](int j) {  // rows j .. j + R - 1 of the 32
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int64_t row = __shfl_sync(0xffffffffu, mine, j + u * RL + rl);
      v[u].zero();
      if (row >= 0 && row < p.n && in) {
        if constexpr (APART)
          v[u].load(dy + row * p.ds, HOP, p.C - c0);
        else
          v[u].load(dy + row * p.ds);
      }  // a row outside the tensor counts as none
    }
  };
  uint32_t b32 = i0;
  auto take = [&](uint32_t b) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
      sum[k] += acc[k];
      acc[k] = 0.f;
    }
    mine = next;
    next = b + 32 + lane < stop ? p.order[b + 32 + lane] : -1;
  };
  while (b32 < stop) {
    // 32 rows of one group
    for (; b32 + 32 <= min(hi, stop); b32 += 32) {
      take(b32);
#pragma unroll 1
      for (int j = 0; j < 32; j += R) {
        load(j);
#pragma unroll
        for (int u = 0; u < UN; ++u) v[u].add_to(acc);
      }
    }
    if (b32 >= stop) break;
    // 32 rows with an end in them
    take(b32);
#pragma unroll 1
    for (uint32_t b = b32; b < min(b32 + 32, stop); b += R) {
      load((int)(b - b32));
      const uint32_t end = min(b + R, stop);
      uint32_t a = b;
      while (true) {
        const uint32_t e = min(hi, end);  // rows [a, e) belong to group g
#pragma unroll
        for (int u = 0; u < UN; ++u) {
          const uint32_t at = b + u * RL + rl;
          if (at >= a && at < e) v[u].add_to(acc);
        }
        if (hi > end || g >= p.G) break;
        flush();  // the group ends here
        a = e;
        do {
          lo = hi;
          hi = ++g < p.G ? offset(g + 1) : UINT32_MAX;
        } while (hi <= a);
        if (a >= end) break;
      }
    }
    b32 += 32;
  }
  if (g < p.G && lo < stop) flush();  // a group that goes on in the next share
}

// The same group by group, for bf16 in 16-byte pieces: the cuts cost their eight sums a lane more than the waits (1.5M
// rows of 64 channels in 7921 groups 58 us so, 65 cut; 1M rows of 128 in 89 groups 59 and 68).
template <typename T, int V, int RL>
__global__ void __launch_bounds__(EG_THREADS, 3) k_embed_grad_by_group(EmbedGrad p) {
  pdl_wait();
  constexpr int CL = 32 / RL;             // channel lanes
  constexpr int UN = RL == 8 ? 4 : 8;     // row loads in flight per lane (UN RL <= 32)
  const int lane = threadIdx.x & 31, cl = lane % CL, rl = lane / CL;
  const int64_t share = blockIdx.x * (int64_t)(EG_THREADS / 32) + (threadIdx.x >> 5);
  if (share >= p.shares) return;
  const int c0 = (blockIdx.y * CL + cl) * V;
  const bool in = c0 < p.C;
  const int64_t i1 = imin64(p.n, (share + 1) * p.share);
  int64_t i = share * p.share;
  const T* dy = static_cast<const T*>(p.dy) + (in ? c0 : 0);
  bool first = true;
  int g = group_at(p.offsets, p.G, i);
  while (i < i1 && g < p.G) {  // (padding rows are last)
    const int64_t lo = p.offsets[g], hi = p.offsets[g + 1];
    const int64_t end = imin64(i1, hi);
    float acc[V] = {};
    // 32 rows of the list at a time; a row outside the tensor counts as none
    int32_t next = i + lane < end ? p.order[i + lane] : -1;
    for (int64_t b = i; b < end; b += 32) {
      const int32_t mine = next;
      next = b + 32 + lane < end ? p.order[b + 32 + lane] : -1;
      const int rows = (int)imin64(32, end - b);
#pragma unroll 1
      for (int j0 = 0; j0 < rows; j0 += UN * RL) {
        Raw<T, V> v[UN];
#pragma unroll
        for (int u = 0; u < UN; ++u) {
          const int j = j0 + u * RL + rl;
          const int64_t row = __shfl_sync(0xffffffffu, mine, j);
          v[u].zero();
          if (row >= 0 && row < p.n && in) v[u].load(dy + row * p.ds);
        }
#pragma unroll
        for (int u = 0; u < UN; ++u) v[u].add_to(acc);
      }
    }
#pragma unroll
    for (int o = CL; o < 32; o <<= 1)
#pragma unroll
      for (int k = 0; k < V; ++k) acc[k] += __shfl_xor_sync(0xffffffffu, acc[k], o);
    if (rl == 0 && in) {
      const bool whole = lo >= share * p.share && hi <= i1;
      if (whole) {
#pragma unroll
        for (int k = 0; k < V; ++k) acc[k] *= p.scale;
        store_channels<T, V>(static_cast<T*>(p.out) + (int64_t)g * p.C + c0, acc);
      } else {
        float* part = p.part + (share * 2 + (first ? 0 : 1)) * p.C + c0;
#pragma unroll
        for (int k = 0; k < V; ++k) part[k] = acc[k];
      }
    }
    first = false;
    i = end > i ? end : i1;  // offsets that do not rise end the walk
    // the next group with rows: mostly the next one
    if (++g < p.G && !(p.offsets[g + 1] > i)) g = group_at(p.offsets, p.G, i);
  }
}

// Groups that several shares hold: their partial rows, in share order; empty
// groups: zero.  A warp takes a group of few shares by itself; the CTA's 32
// warps take the others together.  32 channels and per_cta groups per CTA and round (few groups: one each, so
// that they are joined side by side).
// (1M rows of 128 channels, 4 groups: 86 us, 157 with a warp to each; 89 groups 91 and 98)
constexpr int EJ_ALONE = 16;

template <typename T>
__global__ void __launch_bounds__(1024) k_embed_grad_join(EmbedGrad p, int per_cta) {
  pdl_wait();
  __shared__ float sums[32][33];
  __shared__ uint32_t many;
  const int cl = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.y * 32 + cl;
  T* out = static_cast<T*>(p.out);
  auto span = [&](int g, int64_t* s0, int64_t* s1) -> bool {  // shares of group g; false: empty
    const Range r = group_range(p.offsets, g, p.n);
    if (r.lo >= r.hi) return false;
    *s0 = (uint32_t)r.lo / (uint32_t)p.share;
    *s1 = (uint32_t)(r.hi - 1) / (uint32_t)p.share;
    return true;
  };
  // sum of a group's partial rows from, from + step, ...: this lane's channel
  auto partial = [&](int g, int64_t from, int64_t s0, int64_t s1, int step) -> float {
    float sum = 0.f;
    if (c < p.C)
      for (int64_t s = from; s <= s1;) {
        float acc = 0.f;
#pragma unroll 4
        for (const int64_t e = min(s + 64 * step, s1 + 1); s < e; s += step) {
          // the group is the second of its first share's partial rows unless the share begins with it
          const int which = s > s0 || (int64_t)p.offsets[g] <= s * p.share ? 0 : 1;
          acc += p.part[(s * 2 + which) * p.C + c];
        }
        sum += acc;
      }
    return sum;
  };
  for (int g0 = blockIdx.x * per_cta; g0 < p.G; g0 += gridDim.x * per_cta) {
    if (threadIdx.x == 0) many = 0;
    __syncthreads();
    const int g = g0 + warp;
    int64_t s0 = 0, s1 = 0;
    if (warp < per_cta && g < p.G) {
      if (!span(g, &s0, &s1)) {
        if (c < p.C) out[(int64_t)g * p.C + c] = from_f32<T>(0.f);
      } else if (s1 - s0 >= EJ_ALONE) {
        if (cl == 0) atomicOr(&many, 1u << warp);
      } else if (s1 > s0 && c < p.C) {  // one share: final already
        out[(int64_t)g * p.C + c] = from_f32<T>(p.scale * partial(g, s0, s0, s1, 1));
      }
    }
    __syncthreads();
    for (uint32_t left = many; left; left &= left - 1) {
      const int h = g0 + __ffs(left) - 1;
      span(h, &s0, &s1);
      if (p.C % 4 == 0) {
        // four rows of 32 channels at once, 16 bytes per lane
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        const int quad = blockIdx.y * 32 + (cl & 7) * 4;
        if (quad < p.C) {
#pragma unroll 4
          for (int64_t s = s0 + warp * 4 + (cl >> 3); s <= s1; s += 128) {
            const int which = s > s0 || (int64_t)p.offsets[h] <= s * p.share ? 0 : 1;
            const float4 v = *reinterpret_cast<const float4*>(p.part + (s * 2 + which) * p.C + quad);
            acc.x += v.x;
            acc.y += v.y;
            acc.z += v.z;
            acc.w += v.w;
          }
        }
#pragma unroll
        for (int o = 8; o < 32; o <<= 1) {
          acc.x += __shfl_xor_sync(0xffffffffu, acc.x, o);
          acc.y += __shfl_xor_sync(0xffffffffu, acc.y, o);
          acc.z += __shfl_xor_sync(0xffffffffu, acc.z, o);
          acc.w += __shfl_xor_sync(0xffffffffu, acc.w, o);
        }
        if (cl < 8) {
          sums[warp][cl * 4] = acc.x;
          sums[warp][cl * 4 + 1] = acc.y;
          sums[warp][cl * 4 + 2] = acc.z;
          sums[warp][cl * 4 + 3] = acc.w;
        }
      } else {
        sums[warp][cl] = partial(h, s0 + warp, s0, s1, 32);
      }
      __syncthreads();
      if (warp == 0 && c < p.C) {
        float t = 0.f;
#pragma unroll
        for (int k = 0; k < 32; ++k) t += sums[k][cl];
        out[(int64_t)h * p.C + c] = from_f32<T>(p.scale * t);
      }
      __syncthreads();
    }
  }
}

// scale = max |x| fl(1 / 127) of a row's block, q = x / scale rounded to the nearest: one pass, bound by HBM and by its
// instructions (1.6M rows of 128 fp32 channels 199 us, 5.2 TB/s, with the issue slots 75 % used; bf16 217 us).
// A warp quantises CK_ROWS consecutive (row, block) items, all of their loads in flight; VEC: lane l holds
// channels 4 l .. 4 l + 3 of the block (rows aligned to four channels), else
// channels l, l + 32, l + 64, l + 96.
constexpr int CK_ROWS = 4;

template <typename T, bool VEC>
__global__ void __launch_bounds__(RW_THREADS) k_checkpoint(const T* x, int64_t xn, int64_t xm, int64_t rows, int d,
                                                           int C, int nb, int8_t* q, float* scale) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t items = rows * nb;
  const int64_t i0 = (blockIdx.x * (int64_t)(RW_THREADS / 32) + (threadIdx.x >> 5)) * CK_ROWS;
  if (i0 >= items) return;
  const int here = (int)imin64(CK_ROWS, items - i0);
  // row, node and component of the first item; the others follow by counting
  const int64_t r0 = nb == 1 ? i0 : i0 / nb;
  const int b0 = (int)(i0 - r0 * nb);
  const int64_t node = d == 1 ? r0 : r0 / d;
  const int m0 = (int)(r0 - node * d);
  const int mine_c = VEC ? 4 * lane : lane;  // this lane's first channel of a block
  float v[CK_ROWS][4];
  {
    const T* src = x + node * xn + m0 * xm + mine_c;
    const int64_t wrap = xn - (d - 1) * xm;
    int b = b0, m = m0;
#pragma unroll
    for (int u = 0; u < CK_ROWS; ++u) {
      const int c = b * MACE_CHECKPOINT_BLOCK;
      if constexpr (VEC) {
        v[u][0] = v[u][1] = v[u][2] = v[u][3] = 0.f;
        if (u < here && c + mine_c < C) load4(src + c, v[u]);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[u][j] = u < here && c + mine_c + 32 * j < C ? to_f32(load_in(src + c + 32 * j)) : 0.f;
      }
      if (++b == nb) {
        b = 0;
        if (++m == d) {
          m = 0;
          src += wrap;
        } else {
          src += xm;
        }
      }
    }
  }
  int8_t* dst = q + r0 * C + mine_c;
  int b = b0;
  float mine = 0.f;  // lane u's scale
#pragma unroll
  for (int u = 0; u < CK_ROWS; ++u) {
    // the largest magnitude by its bits: order of floats, with NaN above infinity
    int top = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) top = max(top, __float_as_int(v[u][j]) & 0x7fffffff);
    top = __reduce_max_sync(0xffffffffu, top);
    const float s = __fmul_rn(__int_as_float(top), 1.0f / 127.0f);
    if (lane == u) mine = s;
    const uint32_t packed = quantise8x4(v[u], s);
    const int c = b * MACE_CHECKPOINT_BLOCK;
    if constexpr (VEC) {
      if (u < here && c + mine_c < C) *reinterpret_cast<uint32_t*>(dst + c) = packed;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (u < here && c + mine_c + 32 * j < C) dst[c + 32 * j] = (int8_t)(packed >> (8 * j));
    }
    if (++b == nb) {
      b = 0;
      dst += C;
    }
  }
  if (lane < CK_ROWS && i0 + lane < items) scale[i0 + lane] = mine;
}

// x = q scale, bound by HBM (1.6M rows of 128 fp32 channels 162 us, 6.4 TB/s; bf16 109, 5.7; of 97 channels 166 and 166;
// with 5 CTAs on an SM instead of 8 fp32 183, bf16 151).
// Four consecutive elements of the contiguous (rows, C) result per thread and step; a vector may pass a row's end.
template <typename T>
__global__ void __launch_bounds__(RW_THREADS, 8) k_restore(const int8_t* q, const float* scale, int64_t total, int C, int nb,
                                                        T* x, RowDiv div, int vec) {
  pdl_wait();
  const int64_t e0 = blockIdx.x * (int64_t)(RW_THREADS * RS_UNROLL * 4);
  const int64_t row0 = e0 / C;
  const uint32_t first = (uint32_t)(e0 - row0 * C);
  uint32_t w[RS_UNROLL];
  float sc[RS_UNROLL];  // scale of the vector's first element
#pragma unroll
  for (int j = 0; j < RS_UNROLL; ++j) {
    const int64_t at = e0 + (threadIdx.x + j * RW_THREADS) * 4;
    const uint32_t local = first + (threadIdx.x + j * RW_THREADS) * 4;
    const uint32_t r = div.quotient(local), c = local - r * C;
    w[j] = 0;
    sc[j] = 0.f;
    if (at < total) sc[j] = load_in(scale + (row0 + r) * nb + c / MACE_CHECKPOINT_BLOCK);
    if (vec && at + 4 <= total) {
      w[j] = load_in(reinterpret_cast<const uint32_t*>(q + at));
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (at + k < total) w[j] |= (uint32_t)(uint8_t)load_in(q + at + k) << (8 * k);
    }
  }
  auto values = [&](int j, float* v) {
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = (float)(int8_t)(w[j] >> (8 * k));
  };
  auto store = [&](int j, const float* v) {
    const int64_t at = e0 + (threadIdx.x + j * RW_THREADS) * 4;
    if (vec && at + 4 <= total) {
      store4(x + at, v);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (at + k < total) x[at + k] = from_f32<T>(v[k]);
    }
  };
  if ((C & 3) == 0) {  // a vector has one scale: rows and blocks are multiples of 4
#pragma unroll
    for (int j = 0; j < RS_UNROLL; ++j) {
      float v[4];
      values(j, v);
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] *= sc[j];
      store(j, v);
    }
    return;
  }
  float v[RS_UNROLL][4];
#pragma unroll
  for (int j = 0; j < RS_UNROLL; ++j) {
    const int64_t at = e0 + (threadIdx.x + j * RW_THREADS) * 4;
    values(j, v[j]);
    const uint32_t local = first + (threadIdx.x + j * RW_THREADS) * 4;
    uint32_t r = div.quotient(local), c = local - r * C;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (at + k < total) v[j][k] *= load_in(scale + (row0 + r) * nb + c / MACE_CHECKPOINT_BLOCK);
      if (++c == (uint32_t)C) {
        c = 0;
        ++r;
      }
    }
  }
#pragma unroll
  for (int j = 0; j < RS_UNROLL; ++j) store(j, v[j]);
}

// bits of one counting pass and passes for G + 1 keys
void group_passes(int G, int* bits, int* passes) {
  int b = 1;
  while ((1 << b) < G + 1) ++b;
  *passes = b <= GR_MAX_BITS ? 1 : 2;
  *bits = (b + *passes - 1) / *passes;
}

// rows of one warp's share of the table gradient: enough warps to fill the GPU
// (148 SMs x 3 CTAs x 8 warps) once, or several times over where a share would
// pass 4096 rows (the error of a sum grows with the square root of its terms;
// 20M rows in 1.4 fills instead of 2 take 20 % longer), but at least 16 rows
int64_t eg_share(int64_t n) {
  constexpr int64_t WARPS = 148 * 24;
  const int64_t fills = std::max<int64_t>(1, (n + WARPS * 4096 - 1) / (WARPS * 4096));
  return std::max<int64_t>(16, (n + WARPS * fills - 1) / (WARPS * fills));
}
int64_t eg_shares(int64_t n, int64_t share) { return (n + share - 1) / share; }

int64_t align16(int64_t b) { return (b + 15) & ~(int64_t)15; }

}  // namespace

}  // namespace mace

using namespace mace;

namespace {

// f(std::integral_constant<int, bits>) for 1 <= bits <= MOST
template <int MOST, typename F>
int with_bits(int bits, F&& f) {
  if constexpr (MOST > 1)
    if (bits < MOST) return with_bits<MOST - 1>(bits, f);
  return f(std::integral_constant<int, MOST>{});
}

struct GroupPlan {
  int bits, passes, share, nb;
  bool small;  // one CTA, one launch, no workspace
  int64_t counts, pairs, bytes;  // of the count tables, of the (key, row) pairs between two passes, of all
};
bool group_plan(int64_t n, int32_t G, GroupPlan* p) {
  if (n < 0 || n > INT32_MAX || G < 1 || G > MACE_SPECIES_MAX_INDEX) return false;
  group_passes(G, &p->bits, &p->passes);
  // two rounds of a CTA's warps at least, and no counter of 16 bits overflows
  int64_t step = 0;
  with_bits<GR_MAX_BITS>(p->bits, [&](auto bits) {
    step = GroupCfg<decltype(bits)::value>::THREADS;
    return 0;
  });
  p->share = (int)(std::min(std::max((n + GR_CTAS * step - 1) / (GR_CTAS * step), (int64_t)2), 65535 / step) * step);
  p->nb = (int)((n + p->share - 1) / p->share);
  p->counts = align16(((int64_t)p->nb + 1) * (1 << p->bits) * 4);
  p->pairs = align16(n * 8);
  p->bytes = p->counts + (p->passes > 1 ? p->pairs : 0);
  p->small = n <= GS_MAX_ROWS && G < GS_MAX_BINS;
  if (p->small) p->bytes = 0;
  return true;
}

}  // namespace

extern "C" int mace_species_group_workspace(int64_t n, int32_t G, int64_t* bytes) {
  GroupPlan plan;
  if (!group_plan(n, G, &plan) || !bytes)
    return fail(MACE_ERR_BAD_ARG, "mace_species_group_workspace: bad arguments");
  *bytes = plan.bytes;
  return MACE_OK;
}

extern "C" int mace_species_group(const int32_t* species, int64_t n, int32_t G, int32_t* order, int32_t* offsets,
                                  void* ws, int64_t ws_bytes, void* stream) {
  GroupPlan plan;
  if (!group_plan(n, G, &plan) || !offsets || (n > 0 && (!species || !order)))
    return fail(MACE_ERR_BAD_ARG, "mace_species_group: bad arguments");
  if (unaligned(4, species, order, offsets))
    return fail(MACE_ERR_BAD_ARG, "mace_species_group: an address is not a multiple of its values' size");
  if (plan.bytes > 0 && (!ws || ws_bytes < plan.bytes || (reinterpret_cast<uintptr_t>(ws) & 15) != 0))
    return fail(MACE_ERR_BAD_ARG, "mace_species_group: workspace too small or not 16-byte aligned");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (n == 0) {
    MACE_CUDA_TRY(cudaMemsetAsync(offsets, 0, (size_t)(G + 1) * 4, s));
    return MACE_OK;
  }
  if (plan.small)
    return with_bits<8>(plan.bits, [&](auto bits) {
      return launch("group_small", k_group_small<decltype(bits)::value>, 1, GS_THREADS, 0, s, species, (int)n, G, order,
                    offsets);
    });
  GroupPass p{};
  p.n = n;
  p.G = G;
  p.bits = plan.bits;
  p.share = plan.share;
  p.nb = plan.nb;
  const int bins = 1 << plan.bits;
  char* at = static_cast<char*>(ws);
  p.counts = reinterpret_cast<int32_t*>(at);
  p.totals = p.counts + (int64_t)bins * p.nb;
  int2* const pairs = reinterpret_cast<int2*>(at + plan.counts);
  p.species = species;
  p.order = order;
  for (int q = 0; q < plan.passes; ++q) {
    const bool last = q == plan.passes - 1;
    p.shift = q * plan.bits;
    p.in = q == 0 ? nullptr : pairs;
    p.out = last ? nullptr : pairs;
    p.offsets = plan.passes == 1 ? offsets : nullptr;
    int rc = launch("group_count", k_group_count, p.nb, GR_THREADS, 0, s, p);
    if (!rc) rc = launch("group_scan", k_group_scan, (bins + 31) / 32, GR_THREADS, 0, s, p);
    if (!rc)
      rc = with_bits<GR_MAX_BITS>(plan.bits, [&](auto bits) {
        constexpr int B = decltype(bits)::value;
        static bool attr_set[64] = {};  // per device: the attribute call is slow on the host
        int dev = 0;
        MACE_CUDA_TRY(cudaGetDevice(&dev));
        if (dev >= 64 || !attr_set[dev]) {
          MACE_CUDA_TRY(cudaFuncSetAttribute(k_group_scatter<B>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             GroupCfg<B>::BYTES));
          if (dev < 64) attr_set[dev] = true;
        }
        return launch("group_scatter", k_group_scatter<B>, p.nb, GroupCfg<B>::THREADS, GroupCfg<B>::BYTES, s, p);
      });
    if (rc) return rc;
  }
  if (plan.passes == 1) return MACE_OK;
  return launch("group_offsets", k_group_offsets, (unsigned)(G / 256 + 1), 256, 0, s, species, order, n, G, offsets);
}

namespace {
bool bad_dtype(int32_t t) { return t != MACE_F32 && t != MACE_BF16; }
}  // namespace

namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename T>
int embed(const void* table, int64_t ts, int G, int C, const int32_t* species, int64_t n, float scale, void* out,
          int64_t os, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  const T* t = static_cast<const T*>(table);
  T* o = static_cast<T*>(out);
  auto grid = [&](int v) {
    const int64_t per = (int64_t)RW_THREADS * RW_UNROLL * v;
    return (unsigned)((n * C + per - 1) / per);
  };
  auto go = [&](auto kernel, int v) {
    return launch("species_embed", kernel, grid(v), RW_THREADS, 0, s, t, ts, G, C, species, n, scale, o, os, row_div(C));
  };
  // 1M rows of 128 fp32 channels 77 us (114 as a FLAT result, 215 one by one); of 97 channels 95 FLAT, 164 one by one
  if (!std::isfinite(scale)) return go(k_embed<T, 1, false, true>, 1);
  if (C % V == 0 && ts % V == 0 && os % V == 0 && aligned16(table) && aligned16(out)) return go(k_embed<T, V, false>, V);
  if (os == C && aligned16(out)) return go(k_embed<T, V, true>, V);
  return go(k_embed<T, 1, false>, 1);
}

}  // namespace

extern "C" int mace_species_embed(int32_t dtype, const void* table, int64_t ts, int32_t G, int32_t C,
                                  const int32_t* species, int64_t n, float scale, void* out, int64_t os,
                                  void* stream) {
  if (bad_dtype(dtype) || G < 1 || G > MACE_SPECIES_MAX_INDEX || C < 1 || C > MACE_SPECIES_MAX_CHANNELS ||
      n < 0 || n > INT32_MAX || ts < 0 ||
      !table || (n > 0 && (!species || !out || os < C)))
    return fail(MACE_ERR_BAD_ARG, "mace_species_embed: bad arguments");
  if (unaligned(value_size(dtype), table, out) || unaligned(4, species))
    return fail(MACE_ERR_BAD_ARG, "mace_species_embed: an address is not a multiple of its values' size");
  if (n == 0) return MACE_OK;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return dtype == MACE_F32 ? embed<float>(table, ts, G, C, species, n, scale, out, os, s)
                           : embed<bf16>(table, ts, G, C, species, n, scale, out, os, s);
}

extern "C" int mace_species_embed_grad_workspace(int64_t n, int32_t G, int32_t C, int64_t* bytes) {
  if (n < 0 || n > INT32_MAX || G < 1 || G > MACE_SPECIES_MAX_INDEX || C < 1 ||
      C > MACE_SPECIES_MAX_CHANNELS || !bytes)
    return fail(MACE_ERR_BAD_ARG, "mace_species_embed_grad_workspace: bad arguments");
  *bytes = eg_shares(n, eg_share(n)) * 2 * C * 4;
  return MACE_OK;
}

namespace {

template <typename T, int V>
int launch_embed_grad(const EmbedGrad& p, cudaStream_t s) {
  // row lanes: the most that still leave V channels per lane for one row
  const int cl = (p.C + V - 1) / V;
  const unsigned gx = (unsigned)((p.shares + EG_THREADS / 32 - 1) / (EG_THREADS / 32));
  auto go = [&](auto kernel, int lanes) {
    return launch("species_embed_grad", kernel, dim3(gx, (cl + lanes - 1) / lanes), EG_THREADS, 0, s, p);
  };
  if constexpr (V == 8) {
    if (cl <= 4) return go(k_embed_grad_by_group<T, V, 8>, 4);
    if (cl <= 8) return go(k_embed_grad_by_group<T, V, 4>, 8);
    if (cl <= 16) return go(k_embed_grad_by_group<T, V, 2>, 16);
    return go(k_embed_grad_by_group<T, V, 1>, 32);
  } else {
    // (rows that are not whole pieces: four channels per lane, 32 apart, so that a warp has the row)
    if constexpr (V == 1)
      if (p.C > 32) {
        const dim3 grid(gx, (p.C + 127) / 128);
        return launch("species_embed_grad", k_embed_grad<T, 4, 1, true>, grid, EG_THREADS, 0, s, p);
      }
    if (cl <= 4) return go(k_embed_grad<T, V, 8>, 4);
    if (cl <= 8) return go(k_embed_grad<T, V, 4>, 8);
    if (cl <= 16) return go(k_embed_grad<T, V, 2>, 16);
    return go(k_embed_grad<T, V, 1>, 32);
  }
}

template <typename T>
int embed_grad(const EmbedGrad& p, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  if (p.n > 0) {
    const bool vec = p.C % V == 0 && p.ds % V == 0 && aligned16(p.dy) && aligned16(p.out);
    const int rc = vec ? launch_embed_grad<T, V>(p, s) : launch_embed_grad<T, 1>(p, s);
    if (rc) return rc;
  }
  const int per_cta = std::max(1, std::min(32, (p.G + 147) / 148));
  const dim3 grid(std::min((p.G + per_cta - 1) / per_cta, 148 * 2), (p.C + 31) / 32);
  return launch("species_embed_grad_join", k_embed_grad_join<T>, grid, 1024, 0, s, p, per_cta);
}

}  // namespace

extern "C" int mace_species_embed_grad(int32_t dtype, const void* grad, int64_t gs, const int32_t* order,
                                       const int32_t* offsets, int64_t n, int32_t G, int32_t C, float scale,
                                       void* out, void* ws, int64_t ws_bytes, void* stream) {
  if (bad_dtype(dtype) || n < 0 || n > INT32_MAX || G < 1 || G > MACE_SPECIES_MAX_INDEX || C < 1 ||
      C > MACE_SPECIES_MAX_CHANNELS || gs < 0 || !out ||
      !offsets || (n > 0 && (!grad || !order)))
    return fail(MACE_ERR_BAD_ARG, "mace_species_embed_grad: bad arguments");
  if (unaligned(value_size(dtype), grad, out) || unaligned(4, order, offsets, ws))
    return fail(MACE_ERR_BAD_ARG, "mace_species_embed_grad: an address is not a multiple of its values' size");
  int64_t need = 0;
  mace_species_embed_grad_workspace(n, G, C, &need);
  // (the join reads partial rows four channels at a time)
  if (need > 0 && (!ws || ws_bytes < need || !aligned16(ws)))
    return fail(MACE_ERR_BAD_ARG, "mace_species_embed_grad: workspace too small or not 16-byte aligned");
  EmbedGrad p{grad, gs, order, offsets, n, G, C, eg_share(n), 0, scale, out, static_cast<float*>(ws)};
  p.shares = eg_shares(n, p.share);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return dtype == MACE_F32 ? embed_grad<float>(p, s) : embed_grad<bf16>(p, s);
}

extern "C" int mace_rows_checkpoint(int32_t dtype, const void* x, int64_t xn, int64_t xm, int64_t n, int32_t d,
                                    int32_t C, int8_t* q, float* scale, void* stream) {
  if (bad_dtype(dtype) || n < 0 || n > INT32_MAX || d < 1 || d > 1024 || C < 1 || C > MACE_SPECIES_MAX_CHANNELS || xn < 0 || xm < 0 ||
      (n > 0 && (!x || !q || !scale)))
    return fail(MACE_ERR_BAD_ARG, "mace_rows_checkpoint: bad arguments");
  if (unaligned(value_size(dtype), x) || unaligned(4, scale))
    return fail(MACE_ERR_BAD_ARG, "mace_rows_checkpoint: an address is not a multiple of its values' size");
  if (n == 0) return MACE_OK;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int nb = (C + MACE_CHECKPOINT_BLOCK - 1) / MACE_CHECKPOINT_BLOCK;
  const int64_t per = RW_THREADS / 32 * CK_ROWS;
  const int64_t grid = (n * d * nb + per - 1) / per;
  if (grid > INT32_MAX) return fail(MACE_ERR_BAD_ARG, "mace_rows_checkpoint: too many rows");
  auto go = [&](auto t) {
    using T = decltype(t);
    const T* src = static_cast<const T*>(x);
    const bool vec = C % 4 == 0 && (n <= 1 || xn % 4 == 0) && (d <= 1 || xm % 4 == 0) &&
                     reinterpret_cast<uintptr_t>(x) % (4 * sizeof(T)) == 0 && reinterpret_cast<uintptr_t>(q) % 4 == 0;
    return launch("rows_checkpoint", vec ? k_checkpoint<T, true> : k_checkpoint<T, false>, (unsigned)grid, RW_THREADS, 0,
                  s, src, xn, xm, n * d, d, C, nb, q, scale);
  };
  return dtype == MACE_F32 ? go(float{}) : go(bf16{});
}

extern "C" int mace_rows_restore(int32_t dtype, const int8_t* q, const float* scale, int64_t n, int32_t d, int32_t C,
                                 void* x, void* stream) {
  if (bad_dtype(dtype) || n < 0 || n > INT32_MAX || d < 1 || d > 1024 || C < 1 ||
      C > MACE_SPECIES_MAX_CHANNELS || (n > 0 && (!x || !q || !scale)))
    return fail(MACE_ERR_BAD_ARG, "mace_rows_restore: bad arguments");
  if (unaligned(value_size(dtype), x) || unaligned(4, scale))
    return fail(MACE_ERR_BAD_ARG, "mace_rows_restore: an address is not a multiple of its values' size");
  if (n == 0) return MACE_OK;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int nb = (C + MACE_CHECKPOINT_BLOCK - 1) / MACE_CHECKPOINT_BLOCK;
  const int64_t total = n * d * C, per = RW_THREADS * RS_UNROLL * 4;
  if ((total + per - 1) / per > INT32_MAX) return fail(MACE_ERR_BAD_ARG, "mace_rows_restore: too many rows");
  const unsigned grid = (unsigned)((total + per - 1) / per);
  const int vec = reinterpret_cast<uintptr_t>(q) % 4 == 0 && aligned16(x);
  auto go = [&](auto t) {
    using T = decltype(t);
    return launch("rows_restore", k_restore<T>, grid, RW_THREADS, 0, s, q, scale, total, C, nb, static_cast<T*>(x),
                  row_div(C), vec);
  };
  return dtype == MACE_F32 ? go(float{}) : go(bf16{});
}
