// Gradients of the layer norm (layer_norm.cu) at its rows and parameters.
//
//   dz = dy or dy s (1 + z (1 - s)), s = 1 / (1 + exp(-z)); dw = sum over rows dz xhat, db = sum dz
//   g = w dz, dx = rstd (g - mean(g) - xhat mean(g xhat))
//
// One pass: x and dy stay in registers until dx is stored, and mean and rstd are made once more from the x that has to
// be read anyway, so the forward keeps nothing for it.  A CTA adds the parameters' gradients over its share of the rows
// in registers and leaves one row of sums; a second launch adds those, or, for few rows, the CTAs' own cluster.
#include "layer_norm.cuh"

namespace mace {

namespace {

// column c of (dw, db)
__device__ __forceinline__ void store_param(const LayerNorm& p, int c, float t) {
  void* const out = c < p.C ? p.dw : p.db;
  const int at = c < p.C ? c : c - p.C;
  if (!out) return;
  if (p.param_f32)
    static_cast<float*>(out)[at] = t;
  else
    static_cast<bf16*>(out)[at] = from_f32<bf16>(t);
}

// xhat and dy of a row to dx (in g); the sums of dw and db move on
template <typename T, bool SILU, int N, bool SP, bool SA, typename Sum>
__device__ __forceinline__ void row_grad(const float2* xhat, float2* grad, const Params<N, SP>& params, float rstd,
                                         float inv_C, Sums<N, SA>& acc, Sum& sum) {
  float2 c1 = both(0.f), c2 = both(0.f);
#pragma unroll
  for (int c = 0; c < N / 8; ++c) {
    const float2* const xh = xhat + 4 * c;
    float2 w[4], *const g = grad + 4 * c;
    params.weight(c, w);
    if (SILU) {
      float2 z[4], s[4];
      params.bias(c, z);
#pragma unroll
      for (int i = 0; i < 4; ++i) z[i] = fma2(xh[i], w[i], z[i]);
      sigmoid<T, 4>(z, s);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 rest = fma2(s[i], both(-1.f), both(1.f));
        g[i] = mul2(g[i], mul2(s[i], fma2(z[i], rest, both(1.f))));
      }
    }
    acc.add(c, g, xh);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      g[i] = mul2(g[i], w[i]);
      c1 = add2(c1, g[i]);
      c2 = fma2(g[i], xh[i], c2);
    }
  }
  const float2 c = sum(make_float2(c1.x + c1.y, c2.x + c2.y));
  const float2 m1 = both(-c.x * inv_C), m2 = both(-c.y * inv_C);
#pragma unroll
  for (int i = 0; i < N / 2; ++i) grad[i] = mul2(both(rstd), fma2(xhat[i], m2, add2(grad[i], m1)));
}

// Where a lane keeps its parameters and the sums of their gradients.  Rows of up to 32 lanes: the parameters in shared
// memory, the sums in registers.  Wider ones, whose CTAs the barriers of their sums keep waiting: both in registers
// where rows are whole pieces; else, with the masks, in shared memory, so that four CTAs' threads fit an SM (50 007 rows
// of 1000 105 us, 133 in registers).  (CTAs of more than 256 threads have an SM to themselves.)
template <Layout LAYOUT, int MOST>
constexpr bool LN_WIDE_SHARED = LAYOUT != FULL && MOST == 256;

// Rows of up to 32 lanes: a CTA takes a share of neighbouring rows.  The next row of each lane group is in flight.
template <typename T, Layout LAYOUT, int N, int L, bool SILU>
__global__ void __launch_bounds__(LN_THREADS, 2) k_layer_norm_grad(LayerNorm p) {
  constexpr int GROUPS = LN_THREADS / L, WIDTH = L * N, H = N / 2;
  __shared__ float4 own[2 * N * LN_THREADS / 4];  // the lanes' parameters, in the end the sums
  const int lane = threadIdx.x % L, sub = (threadIdx.x & 31) / L, group = threadIdx.x / L;
  pdl_wait();
  const int64_t begin = blockIdx.x * p.share;
  const uint32_t end = (uint32_t)min(p.n, begin + p.share);
  uint32_t r = (uint32_t)begin + group;
  const T* x = static_cast<const T*>(p.x) + r * p.xs;
  const T* dy = static_cast<const T*>(p.dy) + r * p.ds;
  T* dx = static_cast<T*>(p.y) + r * p.ys;
  const Lane<T, LAYOUT, N> at(lane, L, p.C, LAYOUT == PIECES ? row_head<T>(p.x, p.xs, r) : 0);
  const Params<N, true> params(at, p, own, threadIdx.x, LN_THREADS);
  Sums<N, false> acc(nullptr, threadIdx.x, LN_THREADS);
  Part<T, LAYOUT, N> nx, nd;
  nx.zero();
  nd.zero();
  if (r < end) {
    nx.load(at, x, r - LN_TURN < p.inner);
    nd.load(at, dy, r - LN_TURN < p.inner);
  }
  LaneSum<L> sum;
  __shared__ uint4 edge_slots[LAYOUT == PIECES ? 2 * LN_THREADS / L : 1];
  Edges<T, LAYOUT, N, L> edges(at, p, edge_slots, r, dx);
  for (; r - sub < end; r += GROUPS) {
    float2 v[H], g[H];
    const float lead = nx.template lead<L>();
    nx.values(at, lead, v);
    nd.values(at, 0.f, g);
    x += GROUPS * p.xs;
    dy += GROUPS * p.ds;
    if (r + GROUPS < end) {
      nx.load(at, x, r + GROUPS - LN_TURN < p.inner);
      nd.load(at, dy, r + GROUPS - LN_TURN < p.inner);
    }
    const float rstd = normalise(at, v, lead, p, sum);
    if (r >= end)  // no row
#pragma unroll
      for (int i = 0; i < H; ++i) v[i] = g[i] = both(0.f);
    row_grad<T, SILU>(v, g, params, rstd, p.inv_C, acc, sum);
    if constexpr (LAYOUT == PIECES) {
      if (p.y) {
        edges.store(at, dx, g, r < end, end);
        edges.step(GROUPS, GROUPS * p.ys);
      }
    } else if (p.y && r < end) {
      Part<T, LAYOUT, N>::store(at, dx, g);
    }
    dx += GROUPS * p.ys;
  }
  if (!p.params) return;
  __shared__ float total[2 * WIDTH];
  float* const sums = reinterpret_cast<float*>(own);  // (GROUPS, 2, WIDTH)
  __syncthreads();
#pragma unroll
  for (int j = 0; j < N; ++j)
    if (at.in(j, p.C)) {
      sums[group * 2 * WIDTH + at.at(j)] = acc.get(0, j);
      sums[(group * 2 + 1) * WIDTH + at.at(j)] = acc.get(1, j);
    }
  __syncthreads();
  float* const out = p.part ? p.part + blockIdx.x * (int64_t)p.pitch : total;
  for (int k = threadIdx.x; k < 2 * p.C; k += LN_THREADS) {
    const int which = k >= p.C, c = k - which * p.C;
    float t = 0.f;
#pragma unroll 8
    for (int i = 0; i < GROUPS; ++i) t += sums[(i * 2 + which) * WIDTH + c];
    out[k] = t;
  }
  if (p.part) return;
  cluster_sync();
  for (int k = blockIdx.x * LN_THREADS + threadIdx.x; k < 2 * p.C; k += gridDim.x * LN_THREADS) {
    float t = 0.f;
    for (uint32_t q = 0; q < gridDim.x; ++q) t += load_of_cta(total + k, q);
    store_param(p, k, t);
  }
  cluster_sync();  // (no CTA ends while another reads its sums)
}

// wider rows: a CTA takes every LN_TURN-th row of LN_TURN shares, one at a time
template <typename T, Layout LAYOUT, int N, bool SILU, int MOST>
__global__ void __launch_bounds__(MOST, MOST == 256 ? 2 : 1) k_layer_norm_grad_wide(LayerNorm p) {
  constexpr int H = N / 2;
  constexpr bool SHARED = LN_WIDE_SHARED<LAYOUT, MOST>;
  __shared__ __align__(16) float sums[CtaSum<MOST / 32>::FLOATS];
  extern __shared__ float4 own[];
  pdl_wait();
  const int64_t begin = (blockIdx.x / LN_TURN) * LN_TURN * p.share;
  const uint32_t end = (uint32_t)min(p.n, begin + LN_TURN * p.share);
  uint32_t r = (uint32_t)begin + blockIdx.x % LN_TURN;
  const T* x = static_cast<const T*>(p.x) + r * p.xs;
  const T* dy = static_cast<const T*>(p.dy) + r * p.ds;
  T* dx = static_cast<T*>(p.y) + r * p.ys;
  const Lane<T, LAYOUT, N> at(threadIdx.x, blockDim.x, p.C, LAYOUT == PIECES ? row_head<T>(p.x, p.xs, r) : 0);
  const Params<N, SHARED> params(at, p, own, threadIdx.x, blockDim.x);
  Sums<N, SHARED> acc(own + blockDim.x * 2 * N / 4, threadIdx.x, blockDim.x);
  Part<T, LAYOUT, N> nx, nd;
  nx.zero();
  nd.zero();
  nx.load(at, x, r - LN_TURN < p.inner);
  nd.load(at, dy, r - LN_TURN < p.inner);
  float ahead = to_f32(load_in(x));
  CtaSum<MOST / 32> sum(sums);
  for (; r < end; r += LN_TURN) {
    float2 v[H], g[H];
    const float lead = ahead;
    nx.values(at, lead, v);
    nd.values(at, 0.f, g);
    x += LN_TURN * p.xs;
    dy += LN_TURN * p.ds;
    if (r + LN_TURN < end) {
      nx.load(at, x, r < p.inner);
      nd.load(at, dy, r < p.inner);
      ahead = to_f32(load_in(x));
    }
    const float rstd = normalise(at, v, lead, p, sum);
    row_grad<T, SILU>(v, g, params, rstd, p.inv_C, acc, sum);
    if (p.y) Part<T, LAYOUT, N>::store(at, dx, g);
    dx += LN_TURN * p.ys;
  }
  if (!p.params) return;
  float* const out = p.part + blockIdx.x * (int64_t)p.pitch;
#pragma unroll
  for (int j = 0; j < N; ++j)
    if (at.in(j, p.C)) {
      out[at.at(j)] = acc.get(0, j);
      out[p.C + at.at(j)] = acc.get(1, j);
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
  if (c < 2 * p.C) store_param(p, c, t);
}

// Few rows of up to 32 lanes go to one cluster of up to 16 CTAs, whose sums need no second launch and no workspace: up
// to four steps of a CTA (eight where the rows' starts double their lanes), where both take 5 us on the device (1000 rows of
// 128; 6.7 and 4.6 at twice as many steps), but a call 11.5 us instead of 15.4 on the host.
constexpr int LN_FEW = 4, LN_CLUSTER = MOST_OF_CLUSTER;

// lanes of a row that does not take a CTA: by 8 values without what lies before its start, and the most that any type and
// start give it
int least_lanes(int C) { return std::min(row_lanes(8, C, 0), 32); }
int most_lanes(int C) { return std::min(row_lanes(8, C, 16 / 2 - 1), 32); }
bool few_rows(int64_t n, int C) { return C <= 32 * 8 && n <= LN_CLUSTER * LN_FEW * (LN_THREADS / least_lanes(C)); }

// Rows of a CTA: enough CTAs to fill the GPU, or as many times as many that no lane has more than 256 rows, so that a
// sum's error stays that of a few hundred terms.  From n, C, the lanes of a row (which its alignment decides too) and
// the CTAs of one cluster, 0 where there is none.
int64_t grad_share(int64_t n, int C, int lanes, unsigned cluster) {
  if (lanes > 32) {
    const int64_t ctas = LN_SMS * std::max(1, 512 / row_lanes(LN_WIDE, C, 0));
    return std::min<int64_t>(std::max<int64_t>((n + ctas - 1) / ctas, 1), 256);
  }
  const int64_t rows = LN_THREADS / std::max(lanes, least_lanes(C)), ctas = cluster ? cluster : LN_SMS * 4;
  const int64_t times = std::max<int64_t>((n + ctas * rows * 256 - 1) / (ctas * rows * 256), 1);
  const int64_t share = std::max((n + ctas * times - 1) / (ctas * times), rows);
  return (share + LN_TURN - 1) / LN_TURN * LN_TURN;
}
int64_t grad_shares(int64_t n, int C, int lanes, unsigned cluster) {
  const int64_t share = grad_share(n, C, lanes, cluster);
  if (lanes <= 32) return (n + share - 1) / share;
  const int64_t full = n / (LN_TURN * share);
  return full * LN_TURN + std::min<int64_t>(n - full * LN_TURN * share, LN_TURN);
}
int grad_pitch(int C) { return (2 * C + 3) & ~3; }

template <typename T, Layout LAYOUT, int N, bool SILU>
int backward(const LayerNorm& p, int lanes, cudaStream_t s) {
  const dim3 grid((unsigned)p.shares);
  if constexpr (may_be_wide(LAYOUT, N)) {
    if (lanes > 256)
      return launch("layer_norm_grad", k_layer_norm_grad_wide<T, LAYOUT, N, SILU, MACE_LAYER_NORM_MAX_CHANNELS / N>, grid, lanes,
                    0, s, p);
    if (lanes > 32) {
      const auto kernel = k_layer_norm_grad_wide<T, LAYOUT, N, SILU, 256>;
      constexpr int OF_LANE = LN_WIDE_SHARED<LAYOUT, 256> ? Params<N, true>::BYTES + Sums<N, true>::BYTES : 0;
      static DeviceFlags attr_set;  // per device: the attribute call is slow on the host
      int dev = 0;
      MACE_CUDA_TRY(cudaGetDevice(&dev));
      if (OF_LANE * 256 > 49152 && !attr_set.get(dev)) {
        MACE_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, OF_LANE * 256));
        attr_set.set(dev);
      }
      return launch("layer_norm_grad", kernel, grid, lanes, lanes * OF_LANE, s, p);
    }
  }
  return with_lanes<(N > narrow_values<T, true>(LAYOUT))>(lanes, [&](auto l) {
    const auto kernel = k_layer_norm_grad<T, LAYOUT, N, decltype(l)::value, SILU>;
    if (!p.params || p.part) return launch("layer_norm_grad", kernel, grid, LN_THREADS, 0, s, p);
    static ClusterSizes known;
    unsigned most = 0;
    const int rc = most_of_cluster(kernel, LN_THREADS, known, &most);
    if (rc) return rc;
    LayerNorm q = p;  // (fewer CTAs take larger shares)
    q.share = grad_share(p.n, p.C, lanes, most), q.shares = grad_shares(p.n, p.C, lanes, most);
    const unsigned c = cluster_of((unsigned)q.shares, most);
    return launch_clusters("layer_norm_grad", kernel, c, c, LN_THREADS, 0, s, q);
  });
}

}  // namespace

}  // namespace mace

using namespace mace;

extern "C" int mace_layer_norm_grad_workspace(int64_t n, int32_t C, int64_t* bytes) {
  if (n < 0 || n > INT32_MAX || C < 1 || C > MACE_LAYER_NORM_MAX_CHANNELS || !bytes)
    return fail(MACE_ERR_BAD_ARG, "mace_layer_norm_grad_workspace: bad arguments");
  // (rows of these widths take a warp or a CTA, by their alignment)
  int64_t shares = 0;
  if (C <= 32 * LN_WIDE && !few_rows(n, C)) shares = grad_shares(n, C, most_lanes(C), 0);
  if (C > 32 * LN_APART) shares = std::max(shares, grad_shares(n, C, 64, 0));
  *bytes = shares * grad_pitch(C) * 4;
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
  const Span out{dx, dxs, value_size(dtype), false};
  for (const void* param : {weight, bias})
    if (rows_meet(out, {param, 0, value_size(param_dtype), true}, n, C))
      return fail(MACE_ERR_BAD_ARG, "mace_layer_norm_grad: dx overlaps a parameter");
  if (rows_meet(out, {x, xs, value_size(dtype), false}, n, C) || rows_meet(out, {dy, ds, value_size(dtype), false}, n, C))
    return fail(MACE_ERR_BAD_ARG, "mace_layer_norm_grad: dx overlaps x or dy");
  const bool cluster = params && n > 0 && few_rows(n, C);
  LayerNorm p{};
  p.x = x, p.xs = n > 1 ? xs : 0, p.dy = dy, p.ds = n > 1 ? ds : 0, p.w = weight, p.b = bias;
  p.param_f32 = param_dtype == MACE_F32, p.n = n, p.C = C, p.eps = eps, p.inv_C = 1.f / C, p.inner = inner_rows(n), p.y = dx, p.ys = n > 1 ? dxs : 0;
  p.params = params, p.part = cluster ? nullptr : static_cast<float*>(ws);
  p.pitch = grad_pitch(C), p.dw = dweight, p.db = dbias;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (n > 0 && (params || dx)) {
    auto go = [&](auto t) {
      using T = decltype(t);
      const RowPlan plan = row_plan<T, true>(n, C, {{x, p.xs}, {dy, p.ds}, {dx, p.ys}});
      p.share = grad_share(n, C, plan.lanes, 0), p.shares = grad_shares(n, C, plan.lanes, 0);  // (a cluster: its own)
      return with_plan<T, true>(plan, [&](auto layout, auto values) {
        constexpr Layout LAYOUT = decltype(layout)::value;
        constexpr int N = decltype(values)::value;
        return activation == MACE_ACT_SILU ? backward<T, LAYOUT, N, true>(p, plan.lanes, s)
                                           : backward<T, LAYOUT, N, false>(p, plan.lanes, s);
      });
    };
    const int rc = dtype == MACE_F32 ? go(float{}) : go(bf16{});
    if (rc) return rc;
  }
  if (!params || cluster) return MACE_OK;
  return launch("layer_norm_join", k_layer_norm_join, dim3((unsigned)((p.pitch + 31) / 32)), 1024, 0, s, p);
}
