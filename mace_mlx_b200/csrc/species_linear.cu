// Species-indexed linear map (reference tensor_product.py:1046-1305 with a
// one-hot second input) on rows grouped by species, and its weight gradient:
//   y[r] = alpha x[r] W[g],   dW[g] = alpha sum_{r in g} x[r]^T dy[r].
#include <algorithm>

#include "common.cuh"
#include "species.cuh"

namespace mace {

namespace {

constexpr int ST = 64;   // tile of the products
constexpr int SK = 16;   // summation step

template <typename T>
__global__ void __launch_bounds__(256) k_species_linear(const T* __restrict__ x, int64_t xn, int64_t xm,
                                                        const T* __restrict__ w, int transpose, int G, int K, int M,
                                                        const int32_t* __restrict__ order,
                                                        const int32_t* __restrict__ offsets, int64_t n, int d,
                                                        float alpha, T* __restrict__ y, int64_t yn, int64_t ym) {
  __shared__ float sx[SK][ST + 1], sw[SK][ST + 1];
  // row tile blockIdx.x of the groups' tiles, then of the rows outside them
  int64_t t = blockIdx.x;
  int g = 0;
  Range r{0, 0};
  for (; g < G; ++g) {
    r = group_range(offsets, g, n);
    const int64_t nt = ((r.hi - r.lo) * d + ST - 1) / ST;
    if (t < nt) break;
    t -= nt;
  }
  const int64_t first = g == G ? min(max((int64_t)offsets[0], (int64_t)0), n) : 0;
  if (g == G) {
    const int64_t last = max(min(max((int64_t)offsets[G], (int64_t)0), n), first);
    r.lo = 0;
    r.hi = n - (last - first);
  }
  const int64_t r0 = r.lo * d + t * ST, r1 = r.hi * d;
  if (r0 >= r1) return;
  auto node_of = [&](int64_t row) -> int64_t {
    int64_t at = row / d;
    if (g == G && at >= first) at += n - r.hi;
    const int64_t node = order[at];
    return node >= 0 && node < n ? node : -1;
  };
  const int c0 = blockIdx.y * ST, tid = threadIdx.x;
  float acc[4][4] = {};
  if (g < G) {
    for (int k0 = 0; k0 < K; k0 += SK) {
      for (int i = tid; i < SK * ST; i += 256) {
        const int rr = i / SK, k = k0 + i % SK;
        const int64_t row = r0 + rr;
        const int64_t node = row < r1 && k < K ? node_of(row) : -1;
        sx[i % SK][rr] = node >= 0 ? to_f32(x[node * xn + (row % d) * xm + k]) : 0.f;
      }
      for (int i = tid; i < SK * ST; i += 256) {
        const int kk = i / ST, k = k0 + kk, c = c0 + i % ST;
        float v = 0.f;
        if (k < K && c < M) v = to_f32(w[((int64_t)g * K * M) + (transpose ? (int64_t)c * K + k : (int64_t)k * M + c)]);
        sw[kk][i % ST] = v;
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < SK; ++k)
#pragma unroll
        for (int a = 0; a < 4; ++a)
#pragma unroll
          for (int b = 0; b < 4; ++b) acc[a][b] += sx[k][(tid >> 4) + 16 * a] * sw[k][(tid & 15) + 16 * b];
      __syncthreads();
    }
  }
  for (int a = 0; a < 4; ++a) {
    const int64_t row = r0 + (tid >> 4) + 16 * a;
    const int64_t node = row < r1 ? node_of(row) : -1;
    if (node < 0) continue;
    for (int b = 0; b < 4; ++b) {
      const int c = c0 + (tid & 15) + 16 * b;
      if (c < M) y[node * yn + (row % d) * ym + c] = from_f32<T>(alpha * acc[a][b]);
    }
  }
}

template <typename TX, typename T>
__global__ void __launch_bounds__(256) k_species_wgrad(const TX* __restrict__ x, int64_t xn, int64_t xm,
                                                       const float* __restrict__ xs, const T* __restrict__ dy,
                                                       int64_t yn, int64_t ym, int K, int M,
                                                       const int32_t* __restrict__ order,
                                                       const int32_t* __restrict__ offsets, int64_t n, int d,
                                                       float alpha, T* __restrict__ dw) {
  __shared__ float sx[SK][ST + 1], sy[SK][ST + 1];
  const int g = blockIdx.x, k0 = blockIdx.y * ST, c0 = blockIdx.z * ST, tid = threadIdx.x;
  const int nb = (K + MACE_CHECKPOINT_BLOCK - 1) / MACE_CHECKPOINT_BLOCK;
  const Range r = group_range(offsets, g, n);
  // sums of 16 steps, then their sum: a single accumulator would round once per row
  float acc[4][4] = {}, total[4][4] = {};
  int step = 0;
  for (int64_t base = r.lo * d; base < r.hi * d; base += SK) {
    for (int i = tid; i < SK * ST; i += 256) {
      const int64_t row = base + i / ST;
      const int k = k0 + i % ST, c = c0 + i % ST;
      int64_t node = row < r.hi * d ? order[row / d] : -1;
      if (node >= n) node = -1;
      const int m = (int)(row % d);
      float vx = 0.f, vy = 0.f;
      if (node >= 0 && k < K) {
        vx = to_f32(x[node * xn + m * xm + k]);
        if (xs) vx *= xs[(node * d + m) * nb + k / MACE_CHECKPOINT_BLOCK];
      }
      if (node >= 0 && c < M) vy = to_f32(dy[node * yn + m * ym + c]);
      sx[i / ST][i % ST] = vx;
      sy[i / ST][i % ST] = vy;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < SK; ++k)
#pragma unroll
      for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int b = 0; b < 4; ++b) acc[a][b] += sx[k][(tid >> 4) + 16 * a] * sy[k][(tid & 15) + 16 * b];
    __syncthreads();
    if (++step % 16 == 0 || base + SK >= r.hi * d) {
#pragma unroll
      for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          total[a][b] += acc[a][b];
          acc[a][b] = 0.f;
        }
    }
  }
  for (int a = 0; a < 4; ++a)
    for (int b = 0; b < 4; ++b) {
      const int k = k0 + (tid >> 4) + 16 * a, c = c0 + (tid & 15) + 16 * b;
      if (k < K && c < M) dw[((int64_t)g * K + k) * M + c] = from_f32<T>(alpha * total[a][b]);
    }
}

__device__ int g_species_error;  // TC_ERR_TIMEOUT once a bounded wait gave up

bool bad_sizes(int32_t dtype, int64_t n, int32_t d, int32_t G, int32_t K, int32_t M) {
  return (dtype != MACE_F32 && dtype != MACE_BF16) || n < 0 || n > INT32_MAX || d < 1 || d > 1024 || G < 1 ||
         G > MACE_SPECIES_MAX_GROUPS || K < 1 || K > 65536 || M < 1 || M > 65536;
}

}  // namespace

}  // namespace mace

using namespace mace;

extern "C" int mace_species_linear(int32_t dtype, const void* x, int64_t xn, int64_t xm, const void* w,
                                   int32_t transpose, int32_t G, int32_t K, int32_t M, const int32_t* order,
                                   const int32_t* offsets, int64_t n, int32_t d, float alpha, void* y, int64_t yn,
                                   int64_t ym, void* stream) {
  if (bad_sizes(dtype, n, d, G, K, M) || xn < 0 || xm < 0 || yn < 0 || ym < 0 || !w || !offsets ||
      (n > 0 && (!x || !y || !order)))
    return fail(MACE_ERR_BAD_ARG, "mace_species_linear: bad arguments");
  if (n == 0) return MACE_OK;
  const int64_t tiles = (n * d + ST - 1) / ST + G + 1;
  if (tiles > INT32_MAX) return fail(MACE_ERR_BAD_ARG, "mace_species_linear: too many rows");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const dim3 grid((unsigned)tiles, (M + ST - 1) / ST);
  if (dtype == MACE_F32)
    k_species_linear<float><<<grid, 256, 0, s>>>(static_cast<const float*>(x), xn, xm, static_cast<const float*>(w),
                                                 transpose, G, K, M, order, offsets, n, d, alpha,
                                                 static_cast<float*>(y), yn, ym);
  else
    k_species_linear<bf16><<<grid, 256, 0, s>>>(static_cast<const bf16*>(x), xn, xm, static_cast<const bf16*>(w),
                                                transpose, G, K, M, order, offsets, n, d, alpha,
                                                static_cast<bf16*>(y), yn, ym);
  MACE_LAUNCH_CHECK("species_linear");
  return MACE_OK;
}

extern "C" int mace_species_linear_wgrad_workspace(int64_t n, int32_t d, int32_t G, int32_t K, int32_t M,
                                                   int64_t* bytes) {
  if (bad_sizes(MACE_F32, n, d, G, K, M) || !bytes)
    return fail(MACE_ERR_BAD_ARG, "mace_species_linear_wgrad_workspace: bad arguments");
  *bytes = 0;
  return MACE_OK;
}

extern "C" int mace_species_linear_wgrad(int32_t dtype, const void* x, int64_t xn, int64_t xm, const float* xs,
                                         const void* dy, int64_t yn, int64_t ym, int32_t G, int32_t K, int32_t M,
                                         const int32_t* order, const int32_t* offsets, int64_t n, int32_t d,
                                         float alpha, void* dw, void* ws, int64_t ws_bytes, void* stream) {
  if (bad_sizes(dtype, n, d, G, K, M) || xn < 0 || xm < 0 || yn < 0 || ym < 0 || !dw || !offsets ||
      (n > 0 && (!x || !dy || !order)))
    return fail(MACE_ERR_BAD_ARG, "mace_species_linear_wgrad: bad arguments");
  (void)ws;
  (void)ws_bytes;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const dim3 grid(G, (K + ST - 1) / ST, (M + ST - 1) / ST);
  auto go = [&](auto tx, auto ty) {
    using TX = decltype(tx);
    using T = decltype(ty);
    k_species_wgrad<TX, T><<<grid, 256, 0, s>>>(static_cast<const TX*>(x), xn, xm, xs, static_cast<const T*>(dy), yn,
                                                ym, K, M, order, offsets, n, d, alpha, static_cast<T*>(dw));
  };
  if (xs && dtype == MACE_F32)
    go(int8_t{}, float{});
  else if (xs)
    go(int8_t{}, bf16{});
  else if (dtype == MACE_F32)
    go(float{}, float{});
  else
    go(bf16{}, bf16{});
  MACE_LAUNCH_CHECK("species_wgrad");
  return MACE_OK;
}

extern "C" int mace_species_error_flag(int32_t* flag) {
  if (!flag) return fail(MACE_ERR_BAD_ARG, "mace_species_error_flag: null flag");
  MACE_CUDA_TRY(cudaDeviceSynchronize());
  MACE_CUDA_TRY(cudaMemcpyFromSymbol(flag, g_species_error, 4));
  const int zero = 0;
  MACE_CUDA_TRY(cudaMemcpyToSymbol(g_species_error, &zero, 4));
  return MACE_OK;
}
