// Species operators that move rows: stable grouping by species, the node
// embedding and its table gradient, and the 8-bit row checkpoint
// (species_linear.cu holds the species-indexed linear map).
//
// What they restate (paths in the reference project):
//   node embedding (one-hot linear)  mace_mlx/model.py:373-438
#include <algorithm>

#include "common.cuh"
#include "species.cuh"

namespace mace {

namespace {

constexpr int GR_THREADS = 256;
constexpr int GR_WARPS = GR_THREADS / 32;
constexpr int GR_TILE = 4096;     // rows of one block of a counting pass
constexpr int GR_MAX_BINS = 1024;  // bins of one counting pass

// key of a row: its species, or num_groups for padding rows
__device__ __forceinline__ int row_key(int32_t z, int G) { return (z >= 0 && z < G) ? z : G; }

struct GroupPass {
  const int32_t* key;   // species (first pass) or keys sorted by the lower digit
  const int32_t* row;   // null in the first pass: row i is i
  int64_t n;
  int G;
  int shift, bins;
  int nb;               // blocks
  int32_t* counts;      // (bins, nb)
  int32_t* key_out;     // null in a single pass
  int32_t* row_out;
};

__device__ __forceinline__ int digit_of(const GroupPass& p, int32_t z) { return (row_key(z, p.G) >> p.shift) % p.bins; }

__global__ void __launch_bounds__(GR_THREADS) k_group_count(GroupPass p) {
  __shared__ int hist[GR_MAX_BINS];
  for (int b = threadIdx.x; b < p.bins; b += GR_THREADS) hist[b] = 0;
  __syncthreads();
  const int64_t i0 = (int64_t)blockIdx.x * GR_TILE, i1 = imin64(p.n, i0 + GR_TILE);
  for (int64_t i = i0 + threadIdx.x; i < i1; i += GR_THREADS) atomicAdd(&hist[digit_of(p, p.key[i])], 1);
  __syncthreads();
  for (int b = threadIdx.x; b < p.bins; b += GR_THREADS) p.counts[(int64_t)b * p.nb + blockIdx.x] = hist[b];
}

// exclusive sums of m counts, in place, by one block
__global__ void __launch_bounds__(1024) k_group_scan(int32_t* c, int64_t m) {
  __shared__ int part[1024];
  __shared__ int carry;
  const int t = threadIdx.x;
  if (t == 0) carry = 0;
  __syncthreads();
  for (int64_t base = 0; base < m; base += 1024) {
    const int v = base + t < m ? c[base + t] : 0;
    part[t] = v;
    __syncthreads();
    for (int o = 1; o < 1024; o <<= 1) {
      const int a = t >= o ? part[t - o] : 0;
      __syncthreads();
      part[t] += a;
      __syncthreads();
    }
    if (base + t < m) c[base + t] = carry + part[t] - v;
    __syncthreads();
    if (t == 0) carry += part[1023];
    __syncthreads();
  }
}

__global__ void __launch_bounds__(GR_THREADS) k_group_scatter(GroupPass p) {
  extern __shared__ int whist[];  // (GR_WARPS, bins): next output position of a warp's rows of a digit
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  for (int b = tid; b < GR_WARPS * p.bins; b += GR_THREADS) whist[b] = 0;
  __syncthreads();
  constexpr int SEG = GR_TILE / GR_WARPS;  // consecutive rows of one warp
  const int64_t i0 = (int64_t)blockIdx.x * GR_TILE + warp * SEG, i1 = imin64(p.n, i0 + SEG);
  int* mine = whist + warp * p.bins;
  for (int64_t i = i0 + lane; i < i1; i += 32) atomicAdd(&mine[digit_of(p, p.key[i])], 1);
  __syncthreads();
  for (int b = tid; b < p.bins; b += GR_THREADS) {
    int at = p.counts[(int64_t)b * p.nb + blockIdx.x];
    for (int w = 0; w < GR_WARPS; ++w) {
      const int c = whist[w * p.bins + b];
      whist[w * p.bins + b] = at;
      at += c;
    }
  }
  __syncthreads();
  for (int64_t base = i0; base < i1; base += 32) {
    const int64_t i = base + lane;
    const bool in = i < i1;
    const int32_t z = in ? p.key[i] : 0;
    const int dg = in ? digit_of(p, z) : -1;
    const unsigned same = __match_any_sync(0xffffffffu, dg);
    const int rank = __popc(same & ((1u << lane) - 1));
    int at = 0;
    if (in) at = mine[dg] + rank;
    __syncwarp();
    if (in && rank == 0) mine[dg] += __popc(same);
    __syncwarp();
    if (in) {
      p.row_out[at] = p.row ? p.row[i] : (int32_t)i;
      if (p.key_out) p.key_out[at] = row_key(z, p.G);
    }
  }
}

// offsets[v] = first position whose key is >= v
__global__ void k_group_offsets(const int32_t* __restrict__ order, const int32_t* __restrict__ species, int64_t n, int G,
                                int32_t* __restrict__ offsets) {
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i <= n; i += (int64_t)gridDim.x * blockDim.x) {
    const int prev = i > 0 ? row_key(species[order[i - 1]], G) : -1;
    const int cur = i < n ? row_key(species[order[i]], G) : G;
    for (int v = prev + 1; v <= cur; ++v) offsets[v] = (int32_t)i;
  }
}

template <typename T>
__global__ void k_embed(const T* __restrict__ table, int64_t ts, int G, int C, const int32_t* __restrict__ species,
                        int64_t n, float scale, T* __restrict__ out, int64_t os) {
  const int64_t total = n * C;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / C;
    const int c = (int)(i - r * C);
    const int z = species[r];
    float v = 0.f;
    if (z >= 0 && z < G) v = scale * to_f32(table[z * ts + c]);
    out[r * os + c] = from_f32<T>(v);
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

// group of grouped position i: the largest g with offsets[g] <= i (G: past the last group)
__device__ __forceinline__ int group_at(const int32_t* __restrict__ offsets, int G, int64_t i) {
  int lo = 0, hi = G;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (offsets[mid] <= i)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

constexpr int EG_THREADS = 256;

template <typename T, int V, int RL>
__global__ void __launch_bounds__(EG_THREADS) k_embed_grad(EmbedGrad p) {
  constexpr int CL = 32 / RL;  // channel lanes
  const int lane = threadIdx.x & 31, cl = lane % CL, rl = lane / CL;
  const int64_t share = blockIdx.x * (int64_t)(EG_THREADS / 32) + (threadIdx.x >> 5);
  if (share >= p.shares) return;
  const int c0 = (blockIdx.y * CL + cl) * V;
  const int64_t i1 = imin64(p.n, (share + 1) * p.share);
  int64_t i = share * p.share;
  const T* dy = static_cast<const T*>(p.dy);
  bool first = true;
  while (i < i1) {
    const int g = group_at(p.offsets, p.G, i);
    if (g >= p.G) break;  // padding rows are last
    const int64_t lo = p.offsets[g], hi = p.offsets[g + 1];
    const int64_t end = imin64(i1, hi);
    float acc[V] = {};
    if (c0 < p.C) {
#pragma unroll 4
      for (int64_t r = i + rl; r < end; r += RL) {
        const int64_t row = p.order[r];
        if (row < 0 || row >= p.n) continue;
        float v[V];
        load_channels<T, V>(dy + row * p.ds + c0, v);
#pragma unroll
        for (int k = 0; k < V; ++k) acc[k] += v[k];
      }
    }
#pragma unroll
    for (int o = CL; o < 32; o <<= 1)
#pragma unroll
      for (int k = 0; k < V; ++k) acc[k] += __shfl_xor_sync(0xffffffffu, acc[k], o);
    if (rl == 0 && c0 < p.C) {
      const bool whole = lo >= share * p.share && hi <= i1;
      float* part = p.part + (share * 2 + (first ? 0 : 1)) * p.C;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        if (whole)
          static_cast<T*>(p.out)[(int64_t)g * p.C + c0 + k] = from_f32<T>(p.scale * acc[k]);
        else
          part[c0 + k] = acc[k];
      }
    }
    first = false;
    i = end > i ? end : i1;  // offsets that do not rise end the walk
  }
}

// groups that several shares hold: their partial rows, in share order; empty groups: zero
template <typename T>
__global__ void __launch_bounds__(1024) k_embed_grad_join(EmbedGrad p) {
  __shared__ float sums[32][33];
  const int cl = threadIdx.x & 31, rl = threadIdx.x >> 5;
  const int c = blockIdx.y * 32 + cl;
  T* out = static_cast<T*>(p.out);
  for (int g = blockIdx.x; g < p.G; g += gridDim.x) {
    const Range r = group_range(p.offsets, g, p.n);
    if (r.lo >= r.hi) {
      if (rl == 0 && c < p.C) out[(int64_t)g * p.C + c] = from_f32<T>(0.f);
      continue;
    }
    const int64_t s0 = r.lo / p.share, s1 = (r.hi - 1) / p.share;
    if (s0 == s1) continue;  // final already
    float acc = 0.f;
    if (c < p.C) {
#pragma unroll 4
      for (int64_t s = s0 + rl; s <= s1; s += 32) {
        // a share that the group enters from before it holds its first row there
        const int which = s > s0 || r.lo == s * p.share ? 0 : 1;
        acc += p.part[(s * 2 + which) * p.C + c];
      }
    }
    sums[rl][cl] = acc;
    __syncthreads();
    if (rl == 0 && c < p.C) {
      float t = 0.f;
#pragma unroll
      for (int k = 0; k < 32; ++k) t += sums[k][cl];
      out[(int64_t)g * p.C + c] = from_f32<T>(p.scale * t);
    }
    __syncthreads();
  }
}

template <typename T>
__global__ void k_checkpoint(const T* __restrict__ x, int64_t xn, int64_t xm, int64_t rows, int d, int C, int nb,
                             int8_t* __restrict__ q, float* __restrict__ scale) {
  const int lane = threadIdx.x & 31;
  const int64_t item = blockIdx.x * (int64_t)(blockDim.x >> 5) + (threadIdx.x >> 5);
  if (item >= rows * nb) return;
  const int64_t r = item / nb;
  const int b = (int)(item - r * nb);
  const T* src = x + (r / d) * xn + (r % d) * xm;
  float v[4], top = 0.f;
  bool bad = false;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int c = b * MACE_CHECKPOINT_BLOCK + j * 32 + lane;
    v[j] = c < C ? to_f32(src[c]) : 0.f;
    bad |= v[j] != v[j];
    top = fmaxf(top, fabsf(v[j]));
  }
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (__any_sync(0xffffffffu, bad)) top = __int_as_float(0x7fc00000);
  const float s = __fmul_rn(top, 1.0f / 127.0f);
  if (lane == 0) scale[item] = s;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int c = b * MACE_CHECKPOINT_BLOCK + j * 32 + lane;
    if (c < C) q[r * C + c] = quantise8(v[j], s);
  }
}

template <typename T>
__global__ void k_restore(const int8_t* __restrict__ q, const float* __restrict__ scale, int64_t rows, int C, int nb,
                          T* __restrict__ x) {
  const int64_t total = rows * C;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / C;
    const int c = (int)(i - r * C);
    x[i] = from_f32<T>((float)q[i] * scale[r * nb + c / MACE_CHECKPOINT_BLOCK]);
  }
}

int64_t blocks_for(int64_t items, int per_block, int64_t most) {
  return std::max<int64_t>(1, std::min<int64_t>((items + per_block - 1) / per_block, most));
}

// bits of one counting pass and passes for G + 1 keys
void group_passes(int G, int* bits, int* passes) {
  int b = 1;
  while ((1 << b) < G + 1) ++b;
  *passes = b <= 10 ? 1 : 2;
  *bits = (b + *passes - 1) / *passes;
}

// rows of one warp's share of the table gradient: enough warps to fill the
// GPU (148 SMs x 4 CTAs x 8 warps), but shares of at least 16 rows
int64_t eg_share(int64_t n) { return std::max<int64_t>(16, (n + 148 * 32 - 1) / (148 * 32)); }
int64_t eg_shares(int64_t n, int64_t share) { return (n + share - 1) / share; }

int64_t align16(int64_t b) { return (b + 15) & ~(int64_t)15; }

}  // namespace

}  // namespace mace

using namespace mace;

extern "C" int mace_species_group_workspace(int64_t n, int32_t G, int64_t* bytes) {
  if (n < 0 || n > INT32_MAX || G < 1 || G > MACE_SPECIES_MAX_INDEX || !bytes)
    return fail(MACE_ERR_BAD_ARG, "mace_species_group_workspace: bad arguments");
  int bits, passes;
  group_passes(G, &bits, &passes);
  const int64_t nb = (n + GR_TILE - 1) / GR_TILE;
  *bytes = align16(((int64_t)1 << bits) * nb * 4) + (passes > 1 ? 2 * align16(n * 4) : 0);
  return MACE_OK;
}

extern "C" int mace_species_group(const int32_t* species, int64_t n, int32_t G, int32_t* order, int32_t* offsets,
                                  void* ws, int64_t ws_bytes, void* stream) {
  int64_t need = 0;
  if (mace_species_group_workspace(n, G, &need) != MACE_OK || !offsets || (n > 0 && (!species || !order)))
    return fail(MACE_ERR_BAD_ARG, "mace_species_group: bad arguments");
  if (n > 0 && (!ws || ws_bytes < need)) return fail(MACE_ERR_BAD_ARG, "mace_species_group: workspace too small");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (n == 0) {
    MACE_CUDA_TRY(cudaMemsetAsync(offsets, 0, (size_t)(G + 1) * 4, s));
    return MACE_OK;
  }
  int bits, passes;
  group_passes(G, &bits, &passes);
  GroupPass p{};
  p.n = n;
  p.G = G;
  p.bins = 1 << bits;
  p.nb = (int)((n + GR_TILE - 1) / GR_TILE);
  p.counts = static_cast<int32_t*>(ws);
  int32_t* key2 = reinterpret_cast<int32_t*>(static_cast<char*>(ws) + align16((int64_t)p.bins * p.nb * 4));
  int32_t* row2 = reinterpret_cast<int32_t*>(reinterpret_cast<char*>(key2) + align16(n * 4));
  for (int q = 0; q < passes; ++q) {
    p.shift = q * bits;
    p.key = q == 0 ? species : key2;
    p.row = q == 0 ? nullptr : row2;
    const bool last = q == passes - 1;
    p.key_out = last ? nullptr : key2;
    p.row_out = last ? order : row2;
    k_group_count<<<p.nb, GR_THREADS, 0, s>>>(p);
    MACE_LAUNCH_CHECK("group_count");
    k_group_scan<<<1, 1024, 0, s>>>(p.counts, (int64_t)p.bins * p.nb);
    MACE_LAUNCH_CHECK("group_scan");
    k_group_scatter<<<p.nb, GR_THREADS, GR_WARPS * p.bins * 4, s>>>(p);
    MACE_LAUNCH_CHECK("group_scatter");
  }
  k_group_offsets<<<(int)blocks_for(n + 1, 256, 148 * 8), 256, 0, s>>>(order, species, n, G, offsets);
  MACE_LAUNCH_CHECK("group_offsets");
  return MACE_OK;
}

namespace {
bool bad_dtype(int32_t t) { return t != MACE_F32 && t != MACE_BF16; }
}  // namespace

extern "C" int mace_species_embed(int32_t dtype, const void* table, int64_t ts, int32_t G, int32_t C,
                                  const int32_t* species, int64_t n, float scale, void* out, int64_t os,
                                  void* stream) {
  if (bad_dtype(dtype) || G < 1 || G > MACE_SPECIES_MAX_INDEX || C < 1 || n < 0 || n > INT32_MAX || ts < 0 ||
      !table || (n > 0 && (!species || !out || os < C)))
    return fail(MACE_ERR_BAD_ARG, "mace_species_embed: bad arguments");
  if (n == 0) return MACE_OK;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int grid = (int)blocks_for(n * C, 256, 148 * 16);
  if (dtype == MACE_F32)
    k_embed<float><<<grid, 256, 0, s>>>(static_cast<const float*>(table), ts, G, C, species, n, scale,
                                        static_cast<float*>(out), os);
  else
    k_embed<bf16><<<grid, 256, 0, s>>>(static_cast<const bf16*>(table), ts, G, C, species, n, scale,
                                       static_cast<bf16*>(out), os);
  MACE_LAUNCH_CHECK("species_embed");
  return MACE_OK;
}

extern "C" int mace_species_embed_grad_workspace(int64_t n, int32_t G, int32_t C, int64_t* bytes) {
  if (n < 0 || n > INT32_MAX || G < 1 || G > MACE_SPECIES_MAX_INDEX || C < 1 || !bytes)
    return fail(MACE_ERR_BAD_ARG, "mace_species_embed_grad_workspace: bad arguments");
  *bytes = eg_shares(n, eg_share(n)) * 2 * C * 4;
  return MACE_OK;
}

namespace {

template <typename T, int V>
void launch_embed_grad(const EmbedGrad& p, cudaStream_t s) {
  // row lanes: the most that still leave V channels per lane for one row
  const int cl = (p.C + V - 1) / V;
  const unsigned gx = (unsigned)((p.shares + EG_THREADS / 32 - 1) / (EG_THREADS / 32));
  if (cl <= 4)
    k_embed_grad<T, V, 8><<<dim3(gx, 1), EG_THREADS, 0, s>>>(p);
  else if (cl <= 8)
    k_embed_grad<T, V, 4><<<dim3(gx, 1), EG_THREADS, 0, s>>>(p);
  else if (cl <= 16)
    k_embed_grad<T, V, 2><<<dim3(gx, 1), EG_THREADS, 0, s>>>(p);
  else
    k_embed_grad<T, V, 1><<<dim3(gx, (cl + 31) / 32), EG_THREADS, 0, s>>>(p);
}

template <typename T>
int embed_grad(const EmbedGrad& p, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  if (p.n > 0) {
    if (p.C % V == 0 && p.ds % V == 0 && (reinterpret_cast<uintptr_t>(p.dy) & 15) == 0)
      launch_embed_grad<T, V>(p, s);
    else
      launch_embed_grad<T, 1>(p, s);
    MACE_LAUNCH_CHECK("species_embed_grad");
  }
  k_embed_grad_join<T><<<dim3((unsigned)std::min(p.G, 148 * 8), (p.C + 31) / 32), 1024, 0, s>>>(p);
  MACE_LAUNCH_CHECK("species_embed_grad_join");
  return MACE_OK;
}

}  // namespace

extern "C" int mace_species_embed_grad(int32_t dtype, const void* grad, int64_t gs, const int32_t* order,
                                       const int32_t* offsets, int64_t n, int32_t G, int32_t C, float scale,
                                       void* out, void* ws, int64_t ws_bytes, void* stream) {
  if (bad_dtype(dtype) || n < 0 || n > INT32_MAX || G < 1 || G > MACE_SPECIES_MAX_INDEX || C < 1 || gs < 0 || !out ||
      !offsets || (n > 0 && (!grad || !order)))
    return fail(MACE_ERR_BAD_ARG, "mace_species_embed_grad: bad arguments");
  int64_t need = 0;
  mace_species_embed_grad_workspace(n, G, C, &need);
  if (need > 0 && (!ws || ws_bytes < need))
    return fail(MACE_ERR_BAD_ARG, "mace_species_embed_grad: workspace too small");
  EmbedGrad p{grad, gs, order, offsets, n, G, C, eg_share(n), 0, scale, out, static_cast<float*>(ws)};
  p.shares = eg_shares(n, p.share);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return dtype == MACE_F32 ? embed_grad<float>(p, s) : embed_grad<bf16>(p, s);
}

extern "C" int mace_rows_checkpoint(int32_t dtype, const void* x, int64_t xn, int64_t xm, int64_t n, int32_t d,
                                    int32_t C, int8_t* q, float* scale, void* stream) {
  if (bad_dtype(dtype) || n < 0 || n > INT32_MAX || d < 1 || d > 1024 || C < 1 || xn < 0 || xm < 0 ||
      (n > 0 && (!x || !q || !scale)))
    return fail(MACE_ERR_BAD_ARG, "mace_rows_checkpoint: bad arguments");
  if (n == 0) return MACE_OK;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int nb = (C + MACE_CHECKPOINT_BLOCK - 1) / MACE_CHECKPOINT_BLOCK;
  const int64_t grid = (n * d * nb + 7) / 8;
  if (grid > INT32_MAX) return fail(MACE_ERR_BAD_ARG, "mace_rows_checkpoint: too many rows");
  if (dtype == MACE_F32)
    k_checkpoint<float><<<(int)grid, 256, 0, s>>>(static_cast<const float*>(x), xn, xm, n * d, d, C, nb, q, scale);
  else
    k_checkpoint<bf16><<<(int)grid, 256, 0, s>>>(static_cast<const bf16*>(x), xn, xm, n * d, d, C, nb, q, scale);
  MACE_LAUNCH_CHECK("rows_checkpoint");
  return MACE_OK;
}

extern "C" int mace_rows_restore(int32_t dtype, const int8_t* q, const float* scale, int64_t n, int32_t d, int32_t C,
                                 void* x, void* stream) {
  if (bad_dtype(dtype) || n < 0 || n > INT32_MAX || d < 1 || d > 1024 || C < 1 || (n > 0 && (!x || !q || !scale)))
    return fail(MACE_ERR_BAD_ARG, "mace_rows_restore: bad arguments");
  if (n == 0) return MACE_OK;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int nb = (C + MACE_CHECKPOINT_BLOCK - 1) / MACE_CHECKPOINT_BLOCK;
  const int grid = (int)blocks_for(n * d * C, 256, 148 * 16);
  if (dtype == MACE_F32)
    k_restore<float><<<grid, 256, 0, s>>>(q, scale, n * d, C, nb, static_cast<float*>(x));
  else
    k_restore<bf16><<<grid, 256, 0, s>>>(q, scale, n * d, C, nb, static_cast<bf16*>(x));
  MACE_LAUNCH_CHECK("rows_restore");
  return MACE_OK;
}
