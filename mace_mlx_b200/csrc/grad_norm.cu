// The 2-norm of many tensors taken as one vector, and their clipping to a largest norm: what a training step does to
// the gradients of a model between its backward and its optimiser (the reference has no training path).
//
//   norm = sqrt(sum over all tensors of g^2), out = g min(1, max_norm / (norm + 1e-6))
//
// Squares are exact in fp64 and are summed there, so nothing overflows or vanishes whatever the gradients' scale, and
// the norm is rounded once.  Tensors are cut into 16-byte pieces at 16-byte addresses and the pieces of all tensors
// into tiles; a CTA takes a run of tiles and leaves one sum, and every CTA of the clipping adds the sums itself, in one
// order.  The list of tensors travels as a kernel parameter: no copy to the device, and a captured call keeps it.
#include <algorithm>
#include <cmath>
#include <vector>

#include "common.cuh"
#include "species.cuh"

namespace mace {

namespace {

constexpr int GN_THREADS = 256;
constexpr int GN_UNROLL = 4;                         // pieces of a thread and tile (loads in flight)
constexpr int GN_TILE = GN_THREADS * GN_UNROLL;      // pieces
constexpr int GN_PER_SM = 6;                         // CTAs
constexpr int GN_CTAS = 148 * GN_PER_SM;             // of a launch, at most
constexpr int GN_MAX_TENSORS = 1024;                 // of a launch: kernel parameters hold 32 764 bytes

constexpr uint8_t IN_BF16 = 1, OUT_BF16 = 2, OUT_PIECES = 4;  // OUT_PIECES: a piece's results are aligned to their size

template <int CAP>
struct GradList {
  int count;
  int elsewhere;  // some results go to other tensors
  uint32_t first[CAP + 1];  // first tile of a tensor
  int64_t size[CAP];
  const void* in[CAP];
  void* out[CAP];
  uint8_t type[CAP];
};

// tensor of a tile
template <int CAP>
__device__ __forceinline__ int tensor_of(const GradList<CAP>& list, uint32_t tile) {
  int lo = 0, hi = list.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (list.first[mid] <= tile)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

// A tile of a tensor: its first piece's first value (which may lie before the tensor), and whether all of its pieces lie
// inside.
struct Tile {
  int64_t e;
  bool whole;
};
template <typename T>
__device__ __forceinline__ Tile tile_of(const void* in, int64_t size, uint32_t nth) {
  constexpr int V = 16 / sizeof(T);
  const int64_t e = (int64_t)nth * (GN_TILE * V) - (int64_t)((reinterpret_cast<uintptr_t>(in) & 15) / sizeof(T));
  return {e, e >= 0 && e + GN_TILE * V <= size};
}

// One of this thread's pieces: its values inside the tensor are [max(e, 0), min(e + V, size)).
template <typename T>
struct Piece {
  static constexpr int V = 16 / sizeof(T);
  uint4 raw;
  __device__ __forceinline__ void load(const T* in, const Tile& tile, int64_t size, int u) {
    const int at = (u * GN_THREADS + (int)threadIdx.x) * V;
    if (tile.whole) {
      raw = load_in(reinterpret_cast<const uint4*>(in + tile.e + at));
      return;
    }
    const int64_t e = tile.e + at;
    raw = make_uint4(0, 0, 0, 0);
    if (e >= 0 && e + V <= size) {
      raw = load_in(reinterpret_cast<const uint4*>(in + e));
    } else {
      alignas(16) T t[V];
#pragma unroll
      for (int k = 0; k < V; ++k) t[k] = e + k >= 0 && e + k < size ? load_in(in + e + k) : from_f32<T>(0.f);
      raw = *reinterpret_cast<const uint4*>(t);
    }
  }
  __device__ __forceinline__ void values(float* v) const {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (sizeof(T) == 4) {
        v[k] = __uint_as_float(w[k]);
      } else {
        v[2 * k] = __uint_as_float(w[k] << 16);
        v[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
      }
    }
  }
};

__device__ __forceinline__ double cta_sum(double a, double* buffer) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
  if ((threadIdx.x & 31) == 0) buffer[threadIdx.x >> 5] = a;
  __syncthreads();
  double t = 0.;
  for (int k = 0; k < (int)blockDim.x / 32; ++k) t += buffer[k];
  return t;
}

// 16-bit values without the conversion's pipe (16 lanes a cycle of an SM: 64 % busy, the issue slots 48 %): their bits,
// moved to where fp64 has them, are the value times 2^(127 - 1023) for zeros and subnormals too.  Infinities and NaN come
// out as values from 2^128 on: a CTA whose sum could hold one converts its values.  (71M values 25 us, 22 for the bytes.)
constexpr double GN_BIAS = 0x1p896;
constexpr double GN_SUSPECT = 0x1p255;  // a sum that may hold one

template <typename T, bool EXACT>
__device__ __forceinline__ void add_squares(const void* in, int64_t size, uint32_t nth, double* acc) {
  const Tile tile = tile_of<T>(in, size, nth);
  Piece<T> p[GN_UNROLL];
#pragma unroll
  for (int u = 0; u < GN_UNROLL; ++u) p[u].load(static_cast<const T*>(in), tile, size, u);
#pragma unroll
  for (int u = 0; u < GN_UNROLL; ++u) {
    if constexpr (sizeof(T) == 2 && !EXACT) {
      const uint32_t w[4] = {p[u].raw.x, p[u].raw.y, p[u].raw.z, p[u].raw.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const double lo = __hiloint2double((int)(w[k] << 13 & 0x0fffe000u), 0) * GN_BIAS;
        const double hi = __hiloint2double((int)(w[k] >> 3 & 0x0fffe000u), 0) * GN_BIAS;
        acc[2 * (k & 1)] = fma(lo, lo, acc[2 * (k & 1)]);
        acc[2 * (k & 1) + 1] = fma(hi, hi, acc[2 * (k & 1) + 1]);
      }
    } else {
      float v[Piece<T>::V];
      p[u].values(v);
#pragma unroll
      for (int k = 0; k < Piece<T>::V; ++k) acc[k & 3] = fma((double)v[k], (double)v[k], acc[k & 3]);
    }
  }
}

// a CTA's run of tiles
struct Run {
  uint32_t lo, hi;
};
__device__ __forceinline__ Run run_of(uint32_t tiles) {
  return {(uint32_t)((uint64_t)tiles * blockIdx.x / gridDim.x), (uint32_t)((uint64_t)tiles * (blockIdx.x + 1) / gridDim.x)};
}

template <bool EXACT, int CAP>
__device__ __forceinline__ double sum_of_run(const GradList<CAP>& list, const Run& run, double* buffer) {
  double acc[4] = {0., 0., 0., 0.};
  int t = tensor_of(list, run.lo);
  for (uint32_t tile = run.lo; tile < run.hi; ++tile) {
    while (tile >= list.first[t + 1]) ++t;
    if (list.type[t] & IN_BF16)
      add_squares<bf16, EXACT>(list.in[t], list.size[t], tile - list.first[t], acc);
    else
      add_squares<float, EXACT>(list.in[t], list.size[t], tile - list.first[t], acc);
  }
  return cta_sum((acc[0] + acc[1]) + (acc[2] + acc[3]), buffer);
}

template <int CAP>
__global__ void __launch_bounds__(GN_THREADS, GN_PER_SM) k_grad_squares(const __grid_constant__ GradList<CAP> list, double* part) {
  __shared__ double sums[2][GN_THREADS / 32];
  pdl_wait();
  const Run run = run_of(list.first[list.count]);
  double total = sum_of_run<false>(list, run, sums[0]);
  if (!(total < GN_SUSPECT)) total = sum_of_run<true>(list, run, sums[1]);
  if (threadIdx.x == 0) part[blockIdx.x] = total;
}

// the norm from the CTAs' sums, the same in every CTA of any launch of this many threads
__device__ __forceinline__ double norm_of(const double* part, int parts, double* buffer) {
  double a = 0.;
#pragma unroll 4
  for (int k = threadIdx.x; k < parts; k += blockDim.x) a += part[k];
  return sqrt(cta_sum(a, buffer));
}

__global__ void __launch_bounds__(GN_THREADS) k_grad_norm(const double* part, int parts, float* norm) {
  __shared__ double sums[GN_THREADS / 32];
  pdl_wait();
  const double total = norm_of(part, parts, sums);
  if (threadIdx.x == 0) *norm = (float)total;
}

// eight values of fp32: a whole sector where they are aligned to it
__device__ __forceinline__ void store8(float* dst, const float* v) {
  if ((reinterpret_cast<uintptr_t>(dst) & 31) == 0) {
    asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "f"(v[0]), "f"(v[1]), "f"(v[2]),
                 "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
                 : "memory");
  } else {
    store4(dst, v);
    store4(dst + 4, v + 4);
  }
}

// The factor as one of fp32, or as two whose product it is where it lies below fp32's normal numbers: 2^-126, which only
// moves the exponent of values from 1 on, and the rest.  (Below 2^-252, where the rest is subnormal too, no result reaches
// 2^-123; smaller values come out within two units of 2^-149.)
struct Scale {
  float a, b;
  __device__ __forceinline__ explicit Scale(double factor) {
    const bool two = factor < 0x1p-126;  // (a factor that is NaN stays so)
    a = factor >= 1. ? 1.f : (two ? 0x1p-126f : (float)factor);
    b = two ? (float)(factor * 0x1p126) : 1.f;
  }
  __device__ __forceinline__ bool none() const { return a == 1.f; }
};

template <typename TI, typename TO>
__device__ __forceinline__ void clip_tile(const void* in, void* out, int64_t size, uint32_t nth, bool pieces, const Scale& scale) {
  constexpr int V = Piece<TI>::V;
  const Tile tile = tile_of<TI>(in, size, nth);
  Piece<TI> p[GN_UNROLL];
#pragma unroll
  for (int u = 0; u < GN_UNROLL; ++u) p[u].load(static_cast<const TI*>(in), tile, size, u);
#pragma unroll
  for (int u = 0; u < GN_UNROLL; ++u) {
    float v[V];
    p[u].values(v);
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = v[k] * scale.a * scale.b;
    const int64_t e = tile.e + (u * GN_THREADS + (int)threadIdx.x) * V;
    TO* const dst = static_cast<TO*>(out) + e;
    if (pieces && (tile.whole || (e >= 0 && e + V <= size))) {
      if constexpr (sizeof(TI) == 2 && sizeof(TO) == 2) {
        store_channels<TO, 8>(dst, v);
      } else if constexpr (V == 8) {
        store8(dst, v);
      } else {
        store4(dst, v);
      }
    } else {
#pragma unroll
      for (int k = 0; k < V; ++k)
        if (e + k >= 0 && e + k < size) dst[k] = from_f32<TO>(v[k]);
    }
  }
}

__device__ __forceinline__ Scale scale_of(double max_norm, double norm) { return Scale(max_norm / (norm + 1e-6)); }

// A CTA goes through its run from the end: what the sums read last is still in L2.
template <int CAP>
__device__ __forceinline__ void clip_run(const GradList<CAP>& list, const Run& run, const Scale& scale) {
  if (run.lo >= run.hi || (scale.none() && !list.elsewhere)) return;
  int t = tensor_of(list, run.hi - 1);
  for (uint32_t tile = run.hi; tile-- > run.lo;) {
    while (tile < list.first[t]) --t;
    if (scale.none() && list.out[t] == list.in[t]) continue;
    const uint32_t nth = tile - list.first[t];
    const uint8_t type = list.type[t];
    const bool pieces = type & OUT_PIECES;
    switch (type & (IN_BF16 | OUT_BF16)) {
      case 0: clip_tile<float, float>(list.in[t], list.out[t], list.size[t], nth, pieces, scale); break;
      case IN_BF16: clip_tile<bf16, float>(list.in[t], list.out[t], list.size[t], nth, pieces, scale); break;
      case OUT_BF16: clip_tile<float, bf16>(list.in[t], list.out[t], list.size[t], nth, pieces, scale); break;
      default: clip_tile<bf16, bf16>(list.in[t], list.out[t], list.size[t], nth, pieces, scale);
    }
  }
}

template <int CAP>
__global__ void __launch_bounds__(GN_THREADS, GN_PER_SM) k_grad_clip(const __grid_constant__ GradList<CAP> list, const double* part,
                                                          int parts, double max_norm, float* norm) {
  __shared__ double sums[GN_THREADS / 32];
  pdl_wait();
  const double total = norm_of(part, parts, sums);
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)total;
  clip_run(list, run_of(list.first[list.count]), scale_of(max_norm, total));
}

// Few tiles: one cluster sums and, with max_norm >= 0, clips in one launch (30 tensors of 39 000 values 4.0 us on the
// device, 3.5 in two launches, but a call takes 4 us less on the host: a launch and a workspace).
constexpr int GN_FEW = MACE_GRAD_FEW_TENSORS;
__global__ void __launch_bounds__(GN_THREADS) k_grad_few(const __grid_constant__ GradList<64> list, double max_norm,
                                                         float* norm) {
  __shared__ double sums[2][GN_THREADS / 32], mine;
  pdl_wait();
  const Run run = run_of(list.first[list.count]);
  double total = sum_of_run<false>(list, run, sums[0]);
  if (!(total < GN_SUSPECT)) total = sum_of_run<true>(list, run, sums[1]);
  if (threadIdx.x == 0) mine = total;
  cluster_sync();
  total = 0.;
  for (uint32_t q = 0; q < gridDim.x; ++q) total += load_of_cta(&mine, q);
  total = sqrt(total);
  cluster_sync();  // (no CTA ends, or writes what another has still to read, before all have the sum)
  if (blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)total;
  if (max_norm >= 0.) clip_run(list, run, scale_of(max_norm, total));
}

struct Tensors {
  int32_t count;
  const void* const* in;
  const int64_t* size;
  const int32_t* type;
  void* const* out;  // null: norm only
  const int32_t* out_type;
};

bool bad_type(int32_t t) { return t != MACE_F32 && t != MACE_BF16; }

int64_t values_of(const Tensors& a) {
  int64_t n = 0;
  for (int32_t t = 0; t < a.count; ++t) n += a.size[t];
  return n;
}

int check(const char* who, const Tensors& a, const float* norm, const void* ws, int64_t ws_bytes) {
  const std::string name(who);
  if (a.count < 0 || !norm || (a.count > 0 && (!a.in || !a.size || !a.type))) return fail(MACE_ERR_BAD_ARG, name + ": bad arguments");
  int64_t pieces = 0;
  for (int32_t t = 0; t < a.count; ++t) {
    if (a.size[t] < 0 || a.size[t] > ((int64_t)1 << 40) || bad_type(a.type[t]) || (a.size[t] > 0 && !a.in[t]) ||
        (a.out && (bad_type(a.out_type[t]) || (a.size[t] > 0 && !a.out[t]))))
      return fail(MACE_ERR_BAD_ARG, name + ": bad arguments (tensor " + std::to_string(t) + ")");
    if (unaligned(value_size(a.type[t]), a.in[t]) || (a.out && unaligned(value_size(a.out_type[t]), a.out[t])))
      return fail(MACE_ERR_BAD_ARG, name + ": an address is not a multiple of its values' size");
    pieces += a.size[t] / 4 + GN_TILE + 2;
    if (pieces > ((int64_t)1 << 41)) return fail(MACE_ERR_BAD_ARG, name + ": too many values");
  }
  if (unaligned(4, norm)) return fail(MACE_ERR_BAD_ARG, name + ": an address is not a multiple of its values' size");
  int64_t need = 0;
  mace_grad_norm_workspace(a.count, values_of(a), &need);
  if (need > 0 && (!ws || ws_bytes < need || (reinterpret_cast<uintptr_t>(ws) & 7) != 0))
    return fail(MACE_ERR_BAD_ARG, name + ": workspace too small or not 8-byte aligned");
  return MACE_OK;
}

// an output that overlaps another tensor of the call
bool overlap(const Tensors& a) {
  struct Span {
    uintptr_t lo, hi;
    bool out;
  };
  std::vector<Span> spans;
  spans.reserve(2 * (size_t)a.count);
  for (int32_t t = 0; t < a.count; ++t) {
    if (a.size[t] == 0) continue;
    const uintptr_t in = reinterpret_cast<uintptr_t>(a.in[t]), out = reinterpret_cast<uintptr_t>(a.out[t]);
    spans.push_back({out, out + a.size[t] * value_size(a.out_type[t]), true});
    if (in != out) spans.push_back({in, in + a.size[t] * value_size(a.type[t]), false});
  }
  const auto before = [](const Span& x, const Span& y) { return x.lo < y.lo; };
  if (!std::is_sorted(spans.begin(), spans.end(), before)) std::sort(spans.begin(), spans.end(), before);
  uintptr_t out_end = 0, any_end = 0;
  for (const Span& s : spans) {
    if (s.lo < (s.out ? any_end : out_end)) return true;
    if (s.out) out_end = std::max(out_end, s.hi);
    any_end = std::max(any_end, s.hi);
  }
  return false;
}

// the next tensors of a launch, from `at` on
template <int CAP>
int fill(const Tensors& a, int32_t at, GradList<CAP>* list) {
  int c = 0;
  list->elsewhere = 0;
  uint32_t tiles = 0;
  for (; at < a.count && c < CAP; ++at) {
    if (a.size[at] == 0) continue;
    const int64_t bytes = a.size[at] * value_size(a.type[at]);
    const uint64_t here = ((reinterpret_cast<uintptr_t>(a.in[at]) & 15) + bytes + 16 * GN_TILE - 1) / (16 * GN_TILE);
    uint8_t type = a.type[at] == MACE_BF16 ? IN_BF16 : 0;
    void* out = nullptr;
    if (a.out) {
      out = a.out[at];
      list->elsewhere |= out != a.in[at];
      const int os = value_size(a.out_type[at]), is = value_size(a.type[at]);
      if (a.out_type[at] == MACE_BF16) type |= OUT_BF16;
      // results of the piece that holds the first value begin this many values before it
      const uintptr_t begin = reinterpret_cast<uintptr_t>(out) - (reinterpret_cast<uintptr_t>(a.in[at]) & 15) / is * os;
      if (begin % std::min(16, 16 / is * os) == 0) type |= OUT_PIECES;
    }
    list->first[c] = tiles;
    list->size[c] = a.size[at];
    list->in[c] = a.in[at];
    list->out[c] = out;
    list->type[c] = type;
    tiles += (uint32_t)here;
    ++c;
  }
  list->count = c;
  list->first[c] = tiles;
  return at;
}

unsigned ctas(uint32_t tiles) { return std::min<uint32_t>(tiles, GN_CTAS); }

template <int CAP>
int run(const Tensors& a, double max_norm, float* norm, void* ws, cudaStream_t s) {
  double* const part = static_cast<double*>(ws);
  GradList<CAP> list;
  int parts = 0;
  for (int32_t at = 0; at < a.count;) {
    at = fill(a, at, &list);
    if (list.count == 0) break;
    const unsigned grid = ctas(list.first[list.count]);
    const int rc = launch("grad_squares", k_grad_squares<CAP>, grid, GN_THREADS, 0, s, list, part + parts);
    if (rc) return rc;
    parts += (int)grid;
  }
  if (!a.out || parts == 0) return launch("grad_norm", k_grad_norm, 1, GN_THREADS, 0, s, part, parts, norm);
  const bool once = a.count <= CAP;  // (then the list still holds them)
  bool begin = true;
  for (int32_t at = 0; at < a.count; begin = false) {
    at = once ? a.count : fill(a, at, &list);
    if (list.count == 0) break;
    const int rc = launch("grad_clip", k_grad_clip<CAP>, ctas(list.first[list.count]), GN_THREADS, 0, s, list, part, parts,
                          max_norm, begin ? norm : nullptr);
    if (rc) return rc;
  }
  return MACE_OK;
}

// tensors whose tiles, at any addresses, are at most GN_FEW
bool few_tiles(int64_t count, int64_t values) {
  return count <= GN_FEW && values <= 16 * GN_TILE / 4 * GN_FEW && count * (16 * GN_TILE + 14) + values * 4 <= 16 * GN_TILE * GN_FEW;
}

int run_few(const Tensors& a, double max_norm, float* norm, cudaStream_t s) {
  GradList<64> list;
  fill(a, 0, &list);
  static ClusterSizes known;
  unsigned most = 0;
  const int rc = most_of_cluster(k_grad_few, GN_THREADS, known, &most);
  if (rc) return rc;
  const unsigned c = cluster_of(list.first[list.count], most);
  return launch_clusters("grad_few", k_grad_few, c, c, GN_THREADS, 0, s, list, a.out ? max_norm : -1., norm);
}

// parameters of 2, 8 or 30 KB
int run(const Tensors& a, double max_norm, float* norm, void* ws, cudaStream_t s) {
  if (few_tiles(a.count, values_of(a))) return run_few(a, max_norm, norm, s);
  if (a.count <= 64) return run<64>(a, max_norm, norm, ws, s);
  if (a.count <= 256) return run<256>(a, max_norm, norm, ws, s);
  return run<GN_MAX_TENSORS>(a, max_norm, norm, ws, s);
}

}  // namespace

}  // namespace mace

using namespace mace;

extern "C" int mace_grad_norm_workspace(int32_t count, int64_t values, int64_t* bytes) {
  if (count < 0 || values < 0 || !bytes) return fail(MACE_ERR_BAD_ARG, "mace_grad_norm_workspace: bad arguments");
  *bytes = few_tiles(count, values) ? 0 : ((int64_t)count + GN_MAX_TENSORS - 1) / GN_MAX_TENSORS * GN_CTAS * 8;
  return MACE_OK;
}

extern "C" int mace_grad_norm(int32_t count, const void* const* grads, const int64_t* sizes, const int32_t* dtypes,
                              float* norm, void* ws, int64_t ws_bytes, void* stream) {
  const Tensors a{count, grads, sizes, dtypes, nullptr, nullptr};
  const int rc = check("mace_grad_norm", a, norm, ws, ws_bytes);
  return rc ? rc : run(a, 0., norm, ws, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int mace_grad_clip(int32_t count, const void* const* grads, const int64_t* sizes, const int32_t* dtypes,
                              void* const* out, const int32_t* out_dtypes, double max_norm, float* norm, void* ws,
                              int64_t ws_bytes, void* stream) {
  if (count > 0 && (!out || !out_dtypes)) return fail(MACE_ERR_BAD_ARG, "mace_grad_clip: bad arguments");
  if (!(max_norm >= 0.) || !std::isfinite(max_norm))
    return fail(MACE_ERR_BAD_ARG, "mace_grad_clip: max_norm must be finite and not negative");
  const Tensors a{count, grads, sizes, dtypes, out, out_dtypes};
  int rc = check("mace_grad_clip", a, norm, ws, ws_bytes);
  if (rc) return rc;
  for (int32_t t = 0; t < count; ++t)
    if (sizes[t] > 0 && out[t] == grads[t] && out_dtypes[t] != dtypes[t])
      return fail(MACE_ERR_BAD_ARG, "mace_grad_clip: a tensor clipped in place keeps its type");
  try {
    if (count > 0 && overlap(a)) return fail(MACE_ERR_BAD_ARG, "mace_grad_clip: an output overlaps another tensor");
  } catch (const std::bad_alloc&) {
    return fail(MACE_ERR_BAD_ARG, "mace_grad_clip: too many tensors");
  }
  return run(a, max_norm, norm, ws, reinterpret_cast<cudaStream_t>(stream));
}
