// Layer norm of feature rows, with the SiLU that follows it in the radial MLP of the non-linear interaction block
// (layer_norm_grad.cu holds its gradients).
//
// What it restates (path in the reference project):
//   Linear -> LayerNorm -> SiLU stacks  mace_mlx/radial.py:344-357
//
//   mean = sum x / C, var = sum (x - mean)^2 / C, xhat = (x - mean) rstd, rstd = 1 / sqrt(var + eps)
//   z = w xhat + b, y = z or z / (1 + exp(-z))
//
// One pass: a row stays in registers, 8 or 16 values a lane, between its load and its store.
#include "layer_norm.cuh"

namespace mace {

namespace {

template <typename T, bool SILU, int N, bool SHARED>
__device__ __forceinline__ void affine(float2* v, const Params<N, SHARED>& params) {
#pragma unroll
  for (int c = 0; c < N / 8; ++c) {
    float2 w[4], b[4];
    params.weight(c, w);
    params.bias(c, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[4 * c + i] = fma2(v[4 * c + i], w[i], b[i]);
  }
  if (SILU) {
    float2 s[N / 2];
    sigmoid<T, N / 2>(v, s);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) v[i] = mul2(v[i], s[i]);
  }
}

// CTAs on an SM, and where the lanes keep their parameters.  32 bytes of a row in flight for each lane of three CTAs
// fill the memory's queues (2M fp32 rows of 64 with SiLU 162 us, 173 with four CTAs, 187 with two); rows that start
// anywhere have less in a lane and take four in fp32 (500 003 rows of 96 71 us, 77 with three).  16 values of a lane
// leave no registers for their parameters (2M bf16 rows of 64 with SiLU 89 us, 110 with parameters in registers).
template <typename T, Layout LAYOUT>
constexpr int LN_PER_SM = sizeof(T) == 4 && LAYOUT == PIECES ? 4 : 3;
template <Layout LAYOUT, int N>
constexpr bool LN_SHARED = N == 16 || LAYOUT == PIECES;

// Rows of up to 32 lanes.  The next row of each lane group is in flight.
template <typename T, Layout LAYOUT, int N, int L, bool SILU>
__global__ void __launch_bounds__(LN_THREADS, LN_PER_SM<T, LAYOUT>) k_layer_norm(LayerNorm p) {
  constexpr bool SHARED = LN_SHARED<LAYOUT, N>;
  __shared__ float4 own[SHARED ? Params<N, SHARED>::BYTES / 16 * LN_THREADS : 1];
  const int lane = threadIdx.x % L, sub = (threadIdx.x & 31) / L;
  pdl_wait();
  const uint32_t n = (uint32_t)p.n, step = gridDim.x * (LN_THREADS / L);
  uint32_t r = (blockIdx.x * LN_THREADS + threadIdx.x) / L;
  const T* x = static_cast<const T*>(p.x) + r * p.xs;
  T* y = static_cast<T*>(p.y) + r * p.ys;
  const int64_t x_step = step * p.xs, y_step = step * p.ys;
  const Lane<T, LAYOUT, N> at(lane, L, p.C, LAYOUT == PIECES ? row_head<T>(p.x, p.xs, r) : 0);
  const Params<N, SHARED> params(at, p, own, threadIdx.x, LN_THREADS);
  Part<T, LAYOUT, N> next;
  next.zero();
  if (r < n) next.load(at, x, r - LN_TURN < p.inner);
  LaneSum<L> sum;
  __shared__ uint4 edge_slots[LAYOUT == PIECES ? 2 * LN_THREADS / L : 1];
  Edges<T, LAYOUT, N, L> edges(at, p, edge_slots, r, y);
  for (; r - sub < n; r += step) {
    float2 v[N / 2];
    const float lead = next.template lead<L>();
    next.values(at, lead, v);
    x += x_step;
    if (r + step < n) next.load(at, x, r + step - LN_TURN < p.inner);
    normalise(at, v, lead, p, sum);
    affine<T, SILU>(v, params);
    if constexpr (LAYOUT == PIECES) {
      edges.store(at, y, v, r < n, n);
      edges.step(step, y_step);
    } else if (r < n) {
      Part<T, LAYOUT, N>::store(at, y, v);
    }
    y += y_step;
  }
}

// Wider rows: a CTA each, as many as fit an SM at once.  16-bit rows, with half the bytes for the same barriers, want
// more of them (40 003 rows of 2048 63 us, 71 with 512 threads on an SM), fp32 rows the registers (40 003 rows of 1000
// with SiLU 58 us, 75 with 768).
template <typename T>
constexpr int wide_threads(int most) {  // on an SM, by CTAs of at most 256 or more threads
  return sizeof(T) == 2 ? (most <= 256 ? 768 : 1024) : (most <= 256 ? 512 : most);
}
template <typename T, Layout LAYOUT, int N, bool SILU, int MOST>
__global__ void __launch_bounds__(MOST, wide_threads<T>(MOST) / MOST) k_layer_norm_wide(LayerNorm p) {
  __shared__ __align__(16) float sums[CtaSum<MOST / 32>::FLOATS];
  pdl_wait();
  const uint32_t n = (uint32_t)p.n, step = gridDim.x;
  uint32_t r = blockIdx.x;  // (the grid is a multiple of LN_TURN, or each CTA has one row)
  const T* x = static_cast<const T*>(p.x) + r * p.xs;
  T* y = static_cast<T*>(p.y) + r * p.ys;
  const Lane<T, LAYOUT, N> at(threadIdx.x, blockDim.x, p.C, LAYOUT == PIECES ? row_head<T>(p.x, p.xs, r) : 0);
  const Params<N, false> params(at, p, nullptr, threadIdx.x, blockDim.x);
  Part<T, LAYOUT, N> next;
  next.zero();
  next.load(at, x, r - LN_TURN < p.inner);
  float ahead = to_f32(load_in(x));
  CtaSum<MOST / 32> sum(sums);
  for (; r < n; r += step) {
    float2 v[N / 2];
    const float lead = ahead;
    next.values(at, lead, v);
    x += step * p.xs;
    if (r + step < n) {
      next.load(at, x, r + step - LN_TURN < p.inner);
      ahead = to_f32(load_in(x));
    }
    normalise(at, v, lead, p, sum);
    affine<T, SILU>(v, params);
    Part<T, LAYOUT, N>::store(at, y, v);
    y += step * p.ys;
  }
}

template <typename T, Layout LAYOUT, int N, bool SILU>
int forward(const LayerNorm& p, int lanes, cudaStream_t s) {
  if constexpr (may_be_wide(LAYOUT, N)) {
    if (lanes > 32) {
      constexpr int MOST = MACE_LAYER_NORM_MAX_CHANNELS / N;  // lanes
      const int threads = wide_threads<T>(lanes <= 256 ? 256 : MOST);
      const int64_t grid = std::min<int64_t>(p.n, LN_SMS * std::max(1, threads / lanes) / LN_TURN * LN_TURN);
      auto go = [&](auto kernel) { return launch("layer_norm", kernel, dim3((unsigned)grid), lanes, 0, s, p); };
      return lanes <= 256 ? go(k_layer_norm_wide<T, LAYOUT, N, SILU, 256>) : go(k_layer_norm_wide<T, LAYOUT, N, SILU, MOST>);
    }
  }
  return with_lanes<(N > narrow_values<T, false>(LAYOUT))>(lanes, [&](auto l) {
    constexpr int L = decltype(l)::value;
    const int64_t per = LN_THREADS / L;
    const int64_t grid = std::min<int64_t>((p.n + per - 1) / per, LN_SMS * LN_PER_SM<T, LAYOUT>);
    return launch("layer_norm", k_layer_norm<T, LAYOUT, N, L, SILU>, dim3((unsigned)grid), LN_THREADS, 0, s, p);
  });
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
  const Span out{y, ys, value_size(dtype), false};
  for (const void* param : {weight, bias})
    if (rows_meet(out, {param, 0, value_size(param_dtype), true}, n, C))
      return fail(MACE_ERR_BAD_ARG, "mace_layer_norm: the result overlaps a parameter");
  if (rows_meet(out, {x, xs, value_size(dtype), false}, n, C))
    return fail(MACE_ERR_BAD_ARG, "mace_layer_norm: the result overlaps x");
  if (n == 0) return MACE_OK;
  LayerNorm p{};
  p.x = x, p.xs = n > 1 ? xs : 0, p.w = weight, p.b = bias, p.param_f32 = param_dtype == MACE_F32, p.n = n, p.C = C;
  p.eps = eps, p.inv_C = 1.f / C, p.inner = inner_rows(n), p.y = y, p.ys = n > 1 ? ys : 0;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  auto go = [&](auto t) {
    using T = decltype(t);
    const RowPlan plan = row_plan<T, false>(n, C, {{x, p.xs}, {y, p.ys}});
    return with_plan<T, false>(plan, [&](auto layout, auto values) {
      constexpr Layout LAYOUT = decltype(layout)::value;
      constexpr int N = decltype(values)::value;
      return activation == MACE_ACT_SILU ? forward<T, LAYOUT, N, true>(p, plan.lanes, s)
                                         : forward<T, LAYOUT, N, false>(p, plan.lanes, s);
    });
  };
  return dtype == MACE_F32 ? go(float{}) : go(bf16{});
}
