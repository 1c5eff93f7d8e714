// Layer norm of feature rows, with the SiLU that follows it in the radial MLP of the non-linear interaction block
// (layer_norm_grad.cu holds its gradients).
//
// What it restates (path in the reference project):
//   Linear -> LayerNorm -> SiLU stacks  mace_mlx/radial.py:344-357
//
//   mean = sum x / C, var = sum (x - mean)^2 / C, xhat = (x - mean) rstd, rstd = 1 / sqrt(var + eps)
//   z = w xhat + b, y = z or z / (1 + exp(-z))
//
// One pass: a row stays in registers, 8 values a lane, between its load and its store.
#include "layer_norm.cuh"

namespace mace {

namespace {

template <bool SILU>
__device__ __forceinline__ void affine(float2* v, const float2* w, const float2* b) {
#pragma unroll
  for (int i = 0; i < LN_VALUES / 2; ++i) v[i] = fma2(v[i], w[i], b[i]);
  if (SILU) {
    float2 s[LN_VALUES / 2];
    sigmoid(v, s);
#pragma unroll
    for (int i = 0; i < LN_VALUES / 2; ++i) v[i] = mul2(v[i], s[i]);
  }
}

// CTAs on an SM.  16-byte pieces of fp32 rows fill the memory's queues from three (2M rows of 64 with SiLU 162 us, 174
// with four, 199 with five), 16-bit rows hide their arithmetic behind five (1M rows of 128 91 us, 99 with four).
template <typename T, Layout LAYOUT>
constexpr int LN_PER_SM = LAYOUT == FULL && sizeof(T) == 2 ? 5 : 3;

// Rows of up to 32 lanes.  The next row of each lane group is in flight (a second and third one in flight cost more
// registers than they hide latency: 16-bit rows 117 us instead of 100).
template <typename T, Layout LAYOUT, int L, bool SILU>
__global__ void __launch_bounds__(LN_THREADS, LN_PER_SM<T, LAYOUT>) k_layer_norm(LayerNorm p) {
  constexpr int H = LN_VALUES / 2;
  const int lane = threadIdx.x % L, sub = (threadIdx.x & 31) / L;
  pdl_wait();
  const uint32_t n = (uint32_t)p.n, step = gridDim.x * (LN_THREADS / L);
  uint32_t r = (blockIdx.x * LN_THREADS + threadIdx.x) / L;
  const T* x = static_cast<const T*>(p.x) + r * p.xs;
  T* y = static_cast<T*>(p.y) + r * p.ys;
  const int64_t x_step = step * p.xs, y_step = step * p.ys;
  const Lane<T, LAYOUT> at(lane, L, p.C, LAYOUT == PIECES ? row_head<T>(p.x, p.xs, r) : 0);
  float2 w[H], b[H];
  at.param(p.w, p.param_f32, 1.f, p.C, w);
  at.param(p.b, p.param_f32, 0.f, p.C, b);
  Part<T, LAYOUT> next;
  next.zero();
  if (r < n) next.load(at, x, r - LN_TURN < p.inner);
  LaneSum<L> sum;
  for (; r - sub < n; r += step) {
    float2 v[H];
    next.values(at, v);
    // (PIECES: the second piece is the row's whatever the first one holds)
    const float lead = __shfl_sync(0xffffffffu, v[0].x, LAYOUT == PIECES ? 1 : 0, L);
    x += x_step;
    if (r + step < n) next.load(at, x, r + step - LN_TURN < p.inner);
    normalise(at, v, lead, p, sum);
    affine<SILU>(v, w, b);
    if (r < n) Part<T, LAYOUT>::store(at, y, v);
    y += y_step;
  }
}

// wider rows: a CTA each
template <typename T, Layout LAYOUT, bool SILU, int MOST>
__global__ void __launch_bounds__(MOST) k_layer_norm_wide(LayerNorm p) {
  constexpr int H = LN_VALUES / 2;
  __shared__ __align__(16) float sums[CtaSum<MOST / 32>::FLOATS];
  pdl_wait();
  const uint32_t n = (uint32_t)p.n, step = gridDim.x;
  uint32_t r = blockIdx.x;  // (the grid is a multiple of LN_TURN, or each CTA has one row)
  const T* x = static_cast<const T*>(p.x) + r * p.xs;
  T* y = static_cast<T*>(p.y) + r * p.ys;
  const Lane<T, LAYOUT> at(threadIdx.x, blockDim.x, p.C, LAYOUT == PIECES ? row_head<T>(p.x, p.xs, r) : 0);
  float2 w[H], b[H];
  at.param(p.w, p.param_f32, 1.f, p.C, w);
  at.param(p.b, p.param_f32, 0.f, p.C, b);
  Part<T, LAYOUT> next;
  next.zero();
  next.load(at, x, r - LN_TURN < p.inner);
  float ahead = to_f32(load_in(x));
  CtaSum<MOST / 32> sum(sums);
  for (; r < n; r += step) {
    float2 v[H];
    const float lead = ahead;
    next.values(at, v);
    x += step * p.xs;
    if (r + step < n) {
      next.load(at, x, r + step - LN_TURN < p.inner);
      ahead = to_f32(load_in(x));
    }
    normalise(at, v, lead, p, sum);
    affine<SILU>(v, w, b);
    Part<T, LAYOUT>::store(at, y, v);
    y += step * p.ys;
  }
}

template <typename T, Layout LAYOUT, bool SILU>
int forward(const LayerNorm& p, int lanes, cudaStream_t s) {
  if (lanes > 32) {
    const int64_t grid = std::min<int64_t>(p.n, LN_SMS * std::max(1, 2048 / lanes) / LN_TURN * LN_TURN);
    return launch("layer_norm", lanes <= 256 ? k_layer_norm_wide<T, LAYOUT, SILU, 256> : k_layer_norm_wide<T, LAYOUT, SILU, 1024>,
                  dim3((unsigned)grid), lanes, 0, s, p);
  }
  return with_lanes(lanes, [&](auto l) {
    constexpr int L = decltype(l)::value;
    const int64_t per = LN_THREADS / L;
    const int64_t grid = std::min<int64_t>((p.n + per - 1) / per, LN_SMS * LN_PER_SM<T, LAYOUT>);
    return launch("layer_norm", k_layer_norm<T, LAYOUT, L, SILU>, dim3((unsigned)grid), LN_THREADS, 0, s, p);
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
  if (n == 0) return MACE_OK;
  LayerNorm p{};
  p.x = x, p.xs = n > 1 ? xs : 0, p.w = weight, p.b = bias, p.param_f32 = param_dtype == MACE_F32, p.n = n, p.C = C;
  p.eps = eps, p.inv_C = 1.f / C, p.inner = inner_rows(n), p.y = y, p.ys = n > 1 ? ys : 0;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  auto go = [&](auto t) {
    using T = decltype(t);
    const RowPlan plan = row_plan<T>(n, C, {{x, p.xs}, {y, p.ys}});
    return with_layout(plan.layout, [&](auto layout) {
      constexpr Layout LAYOUT = decltype(layout)::value;
      return activation == MACE_ACT_SILU ? forward<T, LAYOUT, true>(p, plan.lanes, s) : forward<T, LAYOUT, false>(p, plan.lanes, s);
    });
  };
  return dtype == MACE_F32 ? go(float{}) : go(bf16{});
}
