// Layer norm of feature rows, with the SiLU that follows it in the radial MLP of the non-linear interaction block, and
// its gradients.
//
// What it restates (path in the reference project; the reference has no training path):
//   Linear -> LayerNorm -> SiLU stacks  mace_mlx/radial.py:344-357
//
//   forward   mean = sum x / C, var = sum (x - mean)^2 / C, xhat = (x - mean) rstd, rstd = 1 / sqrt(var + eps)
//             z = w xhat + b, y = z or z / (1 + exp(-z))
//   backward  dz = dy or dy s (1 + z (1 - s)), s = 1 / (1 + exp(-z)); dw = sum over rows dz xhat, db = sum dz
//             g = w dz, dx = rstd (g - mean(g) - xhat mean(g xhat))
//
// One pass over the rows each: a row stays in registers, 8 values a lane, between its load and its store, and the
// backward makes mean and rstd once more from the x it has to read anyway, so the forward keeps nothing for it.
#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "species.cuh"

namespace mace {

namespace {

constexpr int LN_THREADS = 256;
constexpr int LN_VALUES = 8;  // of a lane
constexpr int LN_SMS = 148;

struct LayerNorm {
  const void* x;
  int64_t xs;
  const void* dy;
  int64_t ds;
  const void* w;
  const void* b;
  int param_f32;
  int64_t n;
  int C;
  float eps;
  void* y;  // forward: the result; backward: dx, or null
  int64_t ys;
  // backward: rows of a CTA, and its sums: (shares, pitch) with dw in columns [0, C), db behind them
  int64_t share, shares;
  float* part;
  int pitch;
  void* dw;
  void* db;
};

// V consecutive channels per load (a 16-byte piece, or single values): value j of lane `lane` among `lanes` of a row is
// channel ((j / V) lanes + lane) V + j % V
template <typename T, int V>
struct RowPart {
  static constexpr int K = LN_VALUES / V;
  Raw<T, V> raw[K];
  __device__ __forceinline__ void load(const T* row, int lane, int lanes, int C, bool in) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * lanes + lane) * V;
      raw[k].zero();
      if (in && c < C) raw[k].load(row + c);
    }
  }
  __device__ __forceinline__ void values(float* v) const {
#pragma unroll
    for (int k = 0; k < K; ++k) raw[k].values(v + k * V);
  }
  static __device__ __forceinline__ void store(T* row, int lane, int lanes, int C, const float* v) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * lanes + lane) * V;
      if (c < C) store_channels<T, V>(row + c, v + k * V);
    }
  }
};

template <int V>
__device__ __forceinline__ void load_param(const void* p, int f32, float missing, int lane, int lanes, int C, float* v) {
#pragma unroll
  for (int j = 0; j < LN_VALUES; ++j) {
    const int c = ((j / V) * lanes + lane) * V + j % V;
    v[j] = p && c < C ? (f32 ? load_in(static_cast<const float*>(p) + c) : to_f32(load_in(static_cast<const bf16*>(p) + c)))
                      : missing;
  }
}

// sums over the L neighbouring lanes of a row, or over all threads of a CTA
template <int L>
struct LaneSum {
  __device__ __forceinline__ float operator()(float a) const {
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
    return a;
  }
  __device__ __forceinline__ float2 operator()(float2 a) const { return make_float2((*this)(a.x), (*this)(a.y)); }
};
struct CtaSum {
  float2* buffer;  // two of 32 in turn: a thread is past the next barrier only when all have read this one
  int at = 0;
  __device__ __forceinline__ float2 operator()(float2 a) {
    a = LaneSum<32>()(a);
    float2* const b = buffer + at;
    at ^= 32;
    if ((threadIdx.x & 31) == 0) b[threadIdx.x >> 5] = a;
    __syncthreads();
    a = (threadIdx.x & 31) < blockDim.x / 32 ? b[threadIdx.x & 31] : make_float2(0.f, 0.f);
    return LaneSum<32>()(a);
  }
  __device__ __forceinline__ float operator()(float a) { return (*this)(make_float2(a, 0.f)).x; }
};

// A row's values become xhat; rstd is returned.  first: the row's first value.  Sums are taken of x - first: a row of
// equal values comes out as zeros and an offset common to the row costs no accuracy, and first is never further from
// the mean than sqrt(C) standard deviations.
template <int V, typename Sum>
__device__ __forceinline__ float normalise(float* v, float first, int lane, int lanes, int C, float eps, Sum& sum) {
  float a = 0.f;
#pragma unroll
  for (int j = 0; j < LN_VALUES; ++j) {
    const bool on = ((j / V) * lanes + lane) * V < C;
    v[j] = on ? v[j] - first : 0.f;
    a += v[j];
  }
  const float mean = sum(a) / C;
  float q = 0.f;
#pragma unroll
  for (int j = 0; j < LN_VALUES; ++j) {
    const bool on = ((j / V) * lanes + lane) * V < C;
    v[j] = on ? v[j] - mean : 0.f;
    q = fmaf(v[j], v[j], q);
  }
  const float rstd = 1.f / sqrtf(sum(q) / C + eps);
#pragma unroll
  for (int j = 0; j < LN_VALUES; ++j) v[j] *= rstd;
  return rstd;
}

// 1 / (1 + exp(-z)) by CUDA's fast functions: exp within 2 + 1.17 |z| units in the last place, which count where exp(-z)
// outweighs the 1, and the quotient within 2; below z = -87 it may be 0 for 1e-38
__device__ __forceinline__ float sigmoid(float z) { return __fdividef(1.f, 1.f + __expf(-z)); }

template <bool SILU>
__device__ __forceinline__ void affine(float* v, const float* w, const float* b) {
#pragma unroll
  for (int j = 0; j < LN_VALUES; ++j) {
    const float z = fmaf(v[j], w[j], b[j]);
    v[j] = SILU ? z * sigmoid(z) : z;
  }
}

// xhat and dy of a row to dx (in g); sums of dw and db move on
template <bool SILU, bool PARAMS, typename Sum>
__device__ __forceinline__ void row_grad(const float* xhat, float* g, const float* w, const float* b, float rstd, int C,
                                         float* dw, float* db, Sum& sum) {
  float2 c = make_float2(0.f, 0.f);
#pragma unroll
  for (int j = 0; j < LN_VALUES; ++j) {
    if (SILU) {
      const float z = fmaf(xhat[j], w[j], b[j]), s = sigmoid(z);
      g[j] *= s * (1.f + z * (1.f - s));
    }
    if (PARAMS) {
      dw[j] = fmaf(g[j], xhat[j], dw[j]);
      db[j] += g[j];
    }
    g[j] *= w[j];
    c.x += g[j];
    c.y = fmaf(g[j], xhat[j], c.y);
  }
  c = sum(c);
  c.x /= C;
  c.y /= C;
#pragma unroll
  for (int j = 0; j < LN_VALUES; ++j) g[j] = rstd * (g[j] - c.x - xhat[j] * c.y);
}

// rows of up to 256 channels: L lanes each
template <typename T, int V, int L, bool SILU>
__global__ void __launch_bounds__(LN_THREADS) k_layer_norm(LayerNorm p) {
  constexpr int ROWS = 32 / L;
  const int lane = threadIdx.x % L, sub = (threadIdx.x & 31) / L;
  pdl_wait();
  float w[LN_VALUES], b[LN_VALUES];
  load_param<V>(p.w, p.param_f32, 1.f, lane, L, p.C, w);
  load_param<V>(p.b, p.param_f32, 0.f, lane, L, p.C, b);
  const T* const x = static_cast<const T*>(p.x);
  T* const y = static_cast<T*>(p.y);
  const int64_t step = (int64_t)gridDim.x * (LN_THREADS / 32) * ROWS;
  int64_t r = ((int64_t)blockIdx.x * (LN_THREADS / 32) + (threadIdx.x >> 5)) * ROWS + sub;
  RowPart<T, V> next;
  next.load(x + r * p.xs, lane, L, p.C, r < p.n);
  LaneSum<L> sum;
  for (; r - sub < p.n; r += step) {
    float v[LN_VALUES];
    next.values(v);
    next.load(x + (r + step) * p.xs, lane, L, p.C, r + step < p.n);
    const float first = __shfl_sync(0xffffffffu, v[0], 0, L);
    normalise<V>(v, first, lane, L, p.C, p.eps, sum);
    affine<SILU>(v, w, b);
    if (r < p.n) RowPart<T, V>::store(y + r * p.ys, lane, L, p.C, v);
  }
}

// wider rows: a CTA each
template <typename T, int V, bool SILU>
__global__ void __launch_bounds__(1024) k_layer_norm_wide(LayerNorm p) {
  __shared__ float2 sums[64];
  const int lane = threadIdx.x, lanes = blockDim.x;
  pdl_wait();
  float w[LN_VALUES], b[LN_VALUES];
  load_param<V>(p.w, p.param_f32, 1.f, lane, lanes, p.C, w);
  load_param<V>(p.b, p.param_f32, 0.f, lane, lanes, p.C, b);
  const T* const x = static_cast<const T*>(p.x);
  T* const y = static_cast<T*>(p.y);
  RowPart<T, V> next;
  int64_t r = blockIdx.x;
  next.load(x + r * p.xs, lane, lanes, p.C, true);
  float lead = to_f32(load_in(x + r * p.xs));
  CtaSum sum{sums};
  for (; r < p.n; r += gridDim.x) {
    float v[LN_VALUES];
    const float first = lead;
    next.values(v);
    if (r + gridDim.x < p.n) {
      next.load(x + (r + gridDim.x) * p.xs, lane, lanes, p.C, true);
      lead = to_f32(load_in(x + (r + gridDim.x) * p.xs));
    }
    normalise<V>(v, first, lane, lanes, p.C, p.eps, sum);
    affine<SILU>(v, w, b);
    RowPart<T, V>::store(y + r * p.ys, lane, lanes, p.C, v);
  }
}

// gradients of rows of up to 256 channels: a CTA takes a share of the rows and leaves one row of sums
template <typename T, int V, int L, bool SILU, bool PARAMS>
__global__ void __launch_bounds__(LN_THREADS) k_layer_norm_grad(LayerNorm p) {
  constexpr int ROWS = 32 / L, WARPS = LN_THREADS / 32, WIDTH = L * LN_VALUES;
  __shared__ float sums[PARAMS ? WARPS : 1][PARAMS ? 2 * WIDTH : 1];
  const int lane = threadIdx.x % L, sub = (threadIdx.x & 31) / L, warp = threadIdx.x >> 5;
  pdl_wait();
  float w[LN_VALUES], b[LN_VALUES], dw[LN_VALUES], db[LN_VALUES];
  load_param<V>(p.w, p.param_f32, 1.f, lane, L, p.C, w);
  load_param<V>(p.b, p.param_f32, 0.f, lane, L, p.C, b);
#pragma unroll
  for (int j = 0; j < LN_VALUES; ++j) dw[j] = db[j] = 0.f;
  const T* const x = static_cast<const T*>(p.x);
  const T* const dy = static_cast<const T*>(p.dy);
  T* const dx = static_cast<T*>(p.y);
  const int64_t end = min(p.n, (blockIdx.x + 1) * p.share);
  int64_t r = blockIdx.x * p.share + warp * ROWS + sub;
  RowPart<T, V> nx, nd;
  nx.load(x + r * p.xs, lane, L, p.C, r < end);
  nd.load(dy + r * p.ds, lane, L, p.C, r < end);
  LaneSum<L> sum;
  for (; r - sub < end; r += WARPS * ROWS) {
    float v[LN_VALUES], g[LN_VALUES];
    nx.values(v);
    nd.values(g);
    const int64_t to = r + WARPS * ROWS;
    nx.load(x + to * p.xs, lane, L, p.C, to < end);
    nd.load(dy + to * p.ds, lane, L, p.C, to < end);
    const float first = __shfl_sync(0xffffffffu, v[0], 0, L);
    const float rstd = normalise<V>(v, first, lane, L, p.C, p.eps, sum);
    // (a row behind the last is zeros throughout: with eps 0 its xhat is NaN)
    if (r >= end)
#pragma unroll
      for (int j = 0; j < LN_VALUES; ++j) v[j] = 0.f;
    row_grad<SILU, PARAMS>(v, g, w, b, rstd, p.C, dw, db, sum);
    if (dx && r < end) RowPart<T, V>::store(dx + r * p.ys, lane, L, p.C, g);
  }
  if constexpr (PARAMS) {
#pragma unroll
    for (int j = 0; j < LN_VALUES; ++j) {
#pragma unroll
      for (int o = L; o < 32; o <<= 1) {
        dw[j] += __shfl_xor_sync(0xffffffffu, dw[j], o);
        db[j] += __shfl_xor_sync(0xffffffffu, db[j], o);
      }
      const int c = ((j / V) * L + lane) * V + j % V;
      if (sub == 0) {
        sums[warp][c] = dw[j];
        sums[warp][WIDTH + c] = db[j];
      }
    }
    __syncthreads();
    float* const out = p.part + blockIdx.x * (int64_t)p.pitch;
    for (int k = threadIdx.x; k < 2 * WIDTH; k += LN_THREADS) {
      const int c = k % WIDTH;
      float t = 0.f;
#pragma unroll
      for (int i = 0; i < WARPS; ++i) t += sums[i][k];
      if (c < p.C) out[k < WIDTH ? c : p.C + c] = t;
    }
  }
}

// gradients of wider rows: a CTA takes a row at a time of its share
template <typename T, int V, bool SILU, bool PARAMS>
__global__ void __launch_bounds__(1024) k_layer_norm_grad_wide(LayerNorm p) {
  __shared__ float2 sums[64];
  const int lane = threadIdx.x, lanes = blockDim.x;
  pdl_wait();
  float w[LN_VALUES], b[LN_VALUES], dw[LN_VALUES], db[LN_VALUES];
  load_param<V>(p.w, p.param_f32, 1.f, lane, lanes, p.C, w);
  load_param<V>(p.b, p.param_f32, 0.f, lane, lanes, p.C, b);
#pragma unroll
  for (int j = 0; j < LN_VALUES; ++j) dw[j] = db[j] = 0.f;
  const T* const x = static_cast<const T*>(p.x);
  const T* const dy = static_cast<const T*>(p.dy);
  T* const dx = static_cast<T*>(p.y);
  const int64_t end = min(p.n, (blockIdx.x + 1) * p.share);
  int64_t r = blockIdx.x * p.share;
  RowPart<T, V> nx, nd;
  nx.load(x + r * p.xs, lane, lanes, p.C, true);
  nd.load(dy + r * p.ds, lane, lanes, p.C, true);
  float lead = to_f32(load_in(x + r * p.xs));
  CtaSum sum{sums};
  for (; r < end; ++r) {
    float v[LN_VALUES], g[LN_VALUES];
    const float first = lead;
    nx.values(v);
    nd.values(g);
    if (r + 1 < end) {
      nx.load(x + (r + 1) * p.xs, lane, lanes, p.C, true);
      nd.load(dy + (r + 1) * p.ds, lane, lanes, p.C, true);
      lead = to_f32(load_in(x + (r + 1) * p.xs));
    }
    const float rstd = normalise<V>(v, first, lane, lanes, p.C, p.eps, sum);
    row_grad<SILU, PARAMS>(v, g, w, b, rstd, p.C, dw, db, sum);
    if (dx) RowPart<T, V>::store(dx + r * p.ys, lane, lanes, p.C, g);
  }
  if constexpr (PARAMS) {
    float* const out = p.part + blockIdx.x * (int64_t)p.pitch;
#pragma unroll
    for (int j = 0; j < LN_VALUES; ++j) {
      const int c = ((j / V) * lanes + lane) * V + j % V;
      if (c < p.C) {
        out[c] = dw[j];
        out[p.C + c] = db[j];
      }
    }
  }
}

// dw and db from the shares' sums: a CTA adds 32 columns, 4 a lane, a lane group every 128th share
__global__ void __launch_bounds__(1024) k_layer_norm_join(LayerNorm p) {
  __shared__ float4 sums[128][8];
  const int quad = threadIdx.x & 7, slot = threadIdx.x >> 3;
  const int c0 = blockIdx.x * 32 + quad * 4;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  pdl_wait();
  if (c0 < p.pitch) {
#pragma unroll 8
    for (int64_t s = slot; s < p.shares; s += 128) {
      const float4 v = *reinterpret_cast<const float4*>(p.part + s * p.pitch + c0);
      a.x += v.x;
      a.y += v.y;
      a.z += v.z;
      a.w += v.w;
    }
  }
  sums[slot][quad] = a;
  __syncthreads();
  if (threadIdx.x >= 32) return;
  const int c = blockIdx.x * 32 + threadIdx.x;
  float t = 0.f;
#pragma unroll 16
  for (int k = 0; k < 128; ++k) t += reinterpret_cast<const float*>(sums[k])[threadIdx.x];
  if (c >= 2 * p.C) return;
  void* const out = c < p.C ? p.dw : p.db;
  const int at = c < p.C ? c : c - p.C;
  if (!out) return;
  if (p.param_f32)
    static_cast<float*>(out)[at] = t;
  else
    static_cast<bf16*>(out)[at] = from_f32<bf16>(t);
}

// lanes of a row: 8 values each; a power of two up to a warp, then whole warps
int row_lanes(int C) {
  const int need = (C + LN_VALUES - 1) / LN_VALUES;
  if (need > 32) return (need + 31) / 32 * 32;
  int l = 4;
  while (l < need) l *= 2;
  return l;
}

// rows of a CTA of the backward: enough CTAs to fill the GPU, at most 4096 rows, so that a sum's error stays that of
// few hundred terms
int64_t grad_share(int64_t n, int C) {
  const int lanes = row_lanes(C);
  const int64_t rows = lanes > 32 ? 1 : LN_THREADS / lanes;  // at once
  const int64_t ctas = lanes > 32 ? LN_SMS * std::max(1, 1024 / lanes) : LN_SMS * 4;
  int64_t share = std::max((n + ctas - 1) / ctas, rows);
  share = std::min(share, rows * 256);
  return (share + rows - 1) / rows * rows;
}
int grad_pitch(int C) { return (2 * C + 3) & ~3; }

// f(std::integral_constant<int, lanes>) for the lanes of rows of up to 256 channels
template <typename F>
int with_lanes(int lanes, F&& f) {
  switch (lanes) {
    case 4: return f(std::integral_constant<int, 4>{});
    case 8: return f(std::integral_constant<int, 8>{});
    case 16: return f(std::integral_constant<int, 16>{});
    default: return f(std::integral_constant<int, 32>{});
  }
}

template <typename T, int V, bool SILU>
int forward(const LayerNorm& p, cudaStream_t s) {
  const int lanes = row_lanes(p.C);
  if (lanes > 32) {
    const int64_t grid = std::min<int64_t>(p.n, LN_SMS * std::max(1, 2048 / lanes));
    return launch("layer_norm", k_layer_norm_wide<T, V, SILU>, dim3((unsigned)grid), lanes, 0, s, p);
  }
  return with_lanes(lanes, [&](auto l) {
    constexpr int L = decltype(l)::value;
    const int64_t per = LN_THREADS / L;
    const int64_t grid = std::min<int64_t>((p.n + per - 1) / per, LN_SMS * 4);
    return launch("layer_norm", k_layer_norm<T, V, L, SILU>, dim3((unsigned)grid), LN_THREADS, 0, s, p);
  });
}

template <typename T, int V, bool SILU, bool PARAMS>
int backward(const LayerNorm& p, cudaStream_t s) {
  const int lanes = row_lanes(p.C);
  const dim3 grid((unsigned)p.shares);
  if (lanes > 32) return launch("layer_norm_grad", k_layer_norm_grad_wide<T, V, SILU, PARAMS>, grid, lanes, 0, s, p);
  return with_lanes(lanes, [&](auto l) {
    return launch("layer_norm_grad", k_layer_norm_grad<T, V, decltype(l)::value, SILU, PARAMS>, grid, LN_THREADS, 0, s, p);
  });
}

// 16-byte pieces where every row of every operand begins with one and ends with one
template <typename T>
bool whole_pieces(int C, std::initializer_list<const void*> at, std::initializer_list<int64_t> strides) {
  constexpr int V = 16 / sizeof(T);
  bool ok = C % V == 0;
  for (const void* a : at) ok = ok && (reinterpret_cast<uintptr_t>(a) & 15) == 0;
  for (int64_t s : strides) ok = ok && s % V == 0;
  return ok;
}

bool bad_rows(int32_t dtype, int32_t param_dtype, int64_t n, int32_t C, float eps, int32_t activation) {
  return (dtype != MACE_F32 && dtype != MACE_BF16) || (param_dtype != MACE_F32 && param_dtype != MACE_BF16) || n < 0 ||
         n > INT32_MAX || C < 1 || C > MACE_LAYER_NORM_MAX_CHANNELS || !(eps >= 0.f) || !std::isfinite(eps) ||
         (activation != MACE_ACT_NONE && activation != MACE_ACT_SILU);
}

}  // namespace

}  // namespace mace

using namespace mace;

extern "C" int mace_layer_norm(int32_t dtype, const void* x, int64_t xs, int32_t param_dtype, const void* weight,
                               const void* bias, int64_t n, int32_t C, float eps, int32_t activation, void* y,
                               int64_t ys, void* stream) {
  if (bad_rows(dtype, param_dtype, n, C, eps, activation) || xs < 0 || (n > 0 && (!x || !y)) || (n > 1 && ys < C))
    return fail(MACE_ERR_BAD_ARG, "mace_layer_norm: bad arguments");
  if (unaligned(value_size(dtype), x, y) || unaligned(value_size(param_dtype), weight, bias))
    return fail(MACE_ERR_BAD_ARG, "mace_layer_norm: an address is not a multiple of its values' size");
  if (n == 0) return MACE_OK;
  LayerNorm p{};
  p.x = x, p.xs = n > 1 ? xs : 0, p.w = weight, p.b = bias, p.param_f32 = param_dtype == MACE_F32, p.n = n, p.C = C;
  p.eps = eps, p.y = y, p.ys = n > 1 ? ys : 0;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  auto go = [&](auto t) {
    using T = decltype(t);
    constexpr int V = 16 / sizeof(T);
    const bool vec = whole_pieces<T>(C, {x, y}, {p.xs, p.ys});
    if (activation == MACE_ACT_SILU) return vec ? forward<T, V, true>(p, s) : forward<T, 1, true>(p, s);
    return vec ? forward<T, V, false>(p, s) : forward<T, 1, false>(p, s);
  };
  return dtype == MACE_F32 ? go(float{}) : go(bf16{});
}

extern "C" int mace_layer_norm_grad_workspace(int64_t n, int32_t C, int64_t* bytes) {
  if (n < 0 || n > INT32_MAX || C < 1 || C > MACE_LAYER_NORM_MAX_CHANNELS || !bytes)
    return fail(MACE_ERR_BAD_ARG, "mace_layer_norm_grad_workspace: bad arguments");
  const int64_t share = grad_share(n, C);
  *bytes = (n + share - 1) / share * grad_pitch(C) * 4;
  return MACE_OK;
}

extern "C" int mace_layer_norm_grad(int32_t dtype, const void* x, int64_t xs, const void* dy, int64_t ds,
                                    int32_t param_dtype, const void* weight, const void* bias, int64_t n, int32_t C,
                                    float eps, int32_t activation, void* dx, int64_t dxs, void* dweight, void* dbias,
                                    void* ws, int64_t ws_bytes, void* stream) {
  if (bad_rows(dtype, param_dtype, n, C, eps, activation) || xs < 0 || ds < 0 || (n > 0 && (!x || !dy)) ||
      (dx && n > 1 && dxs < C))
    return fail(MACE_ERR_BAD_ARG, "mace_layer_norm_grad: bad arguments");
  if (unaligned(value_size(dtype), x, dy, dx) || unaligned(value_size(param_dtype), weight, bias, dweight, dbias))
    return fail(MACE_ERR_BAD_ARG, "mace_layer_norm_grad: an address is not a multiple of its values' size");
  const bool params = dweight || dbias;
  int64_t need = 0;
  mace_layer_norm_grad_workspace(n, C, &need);
  if (params && need > 0 && (!ws || ws_bytes < need || (reinterpret_cast<uintptr_t>(ws) & 15) != 0))
    return fail(MACE_ERR_BAD_ARG, "mace_layer_norm_grad: workspace too small or not 16-byte aligned");
  LayerNorm p{};
  p.x = x, p.xs = n > 1 ? xs : 0, p.dy = dy, p.ds = n > 1 ? ds : 0, p.w = weight, p.b = bias;
  p.param_f32 = param_dtype == MACE_F32, p.n = n, p.C = C, p.eps = eps, p.y = dx, p.ys = n > 1 ? dxs : 0;
  p.share = grad_share(n, C), p.shares = (n + p.share - 1) / p.share, p.part = static_cast<float*>(ws);
  p.pitch = grad_pitch(C), p.dw = dweight, p.db = dbias;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (n > 0 && (params || dx)) {
    auto go = [&](auto t) {
      using T = decltype(t);
      constexpr int V = 16 / sizeof(T);
      const bool vec = whole_pieces<T>(C, {x, dy, dx}, {p.xs, p.ds, dx ? p.ys : 0});
      auto with = [&](auto v) {
        constexpr int W = decltype(v)::value;
        if (activation == MACE_ACT_SILU) return params ? backward<T, W, true, true>(p, s) : backward<T, W, true, false>(p, s);
        return params ? backward<T, W, false, true>(p, s) : backward<T, W, false, false>(p, s);
      };
      return vec ? with(std::integral_constant<int, V>{}) : with(std::integral_constant<int, 1>{});
    };
    const int rc = dtype == MACE_F32 ? go(float{}) : go(bf16{});
    if (rc) return rc;
  }
  if (!params) return MACE_OK;
  return launch("layer_norm_join", k_layer_norm_join, dim3((unsigned)((p.pitch + 31) / 32)), 1024, 0, s, p);
}
