// Rows of the layer norm in registers (layer_norm.cu, layer_norm_grad.cu): how a row is spread over its lanes, and the
// arithmetic on a lane's values, two at a time (the packed fp32 instructions of sm_100).
#pragma once

#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <numeric>

#include "common.cuh"
#include "species.cuh"

namespace mace {

constexpr int LN_THREADS = 256;  // of a CTA whose rows have up to 32 lanes
constexpr int LN_SMS = 148;
constexpr int LN_TURN = 8;       // rows that many apart begin at the same address modulo 16

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
  float eps, inv_C;
  uint32_t inner;  // rows [LN_TURN, LN_TURN + inner) have LN_TURN neighbours on either side
  void* y;  // forward: the result; backward: dx, or null
  int64_t ys;
  // backward: rows of a CTA, and its sums: (shares, pitch) with dw in columns [0, C), db behind them
  int64_t share, shares;
  bool params;  // dw or db is wanted
  float* part;  // null: the CTAs are one cluster, which adds them itself
  int pitch;
  void* dw;
  void* db;
};

// How a row's channels reach its lanes, N each:
//   FULL    16-byte pieces, every row starts with one, and the lanes take exactly C channels
//   PIECES  16-byte pieces at 16-byte addresses, wherever the row starts: its first and last piece may hold values of
//           its neighbours, which are masked.  A row's start modulo 16 repeats every LN_TURN rows, so lanes that step
//           by that many rows keep their channels.  More channels than a piece has.
//   APART   single values, neighbouring lanes neighbouring channels: rows that start differently modulo 16 in two
//           operands, or that are no longer than a piece
enum Layout { FULL, PIECES, APART };

// ---- two fp32 values at a time
__device__ __forceinline__ uint64_t pack2(float2 a) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a.x), "f"(a.y));
  return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t r) {
  float2 a;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a.x), "=f"(a.y) : "l"(r));
  return a;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pack2(a)), "l"(pack2(b)));
  return unpack2(r);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pack2(a)), "l"(pack2(b)));
  return unpack2(r);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(pack2(a)), "l"(pack2(b)), "l"(pack2(c)));
  return unpack2(r);
}
__device__ __forceinline__ float2 both(float a) { return make_float2(a, a); }
// A lane's channels: value j is channel at(j), and in the row where 0 <= at(j) < C.
template <typename T, Layout LAYOUT, int N>
struct Lane {
  static constexpr int V = LAYOUT == APART ? 1 : 16 / sizeof(T), K = N / V;
  // the bits of a lane's values that are the row's, in words as they lie in memory (APART: of 32 bits each)
  static constexpr int WORDS = LAYOUT == FULL ? 1 : (LAYOUT == PIECES ? N * sizeof(T) / 4 : N);
  int first[K];  // channel of a piece's first value
  int count[K];  // channels of the row in a piece
  uint32_t keep[WORDS];
  static constexpr bool BY_PIECE = LAYOUT == PIECES && sizeof(T) == 4;
  float has[BY_PIECE ? K : 1];  // 1 for a piece that has a value of the row, 0 for others
  float off;     // values of the lane that are not the row's (BY_PIECE: in pieces that have one)
  bool some;     // or all are
  // head: values between a 16-byte address and the row's start
  __device__ __forceinline__ Lane(int lane, int lanes, int C, int head) {
    int all = 0, others = 0;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      first[k] = (k * lanes + lane) * V - head;
      count[k] = LAYOUT == FULL ? V : max(0, min(first[k] + V, C) - max(first[k], 0));
      all += count[k];
      if constexpr (BY_PIECE) {
        has[k] = any(k) ? 1.f : 0.f;
        if (any(k)) others += V - count[k];
      }
    }
    off = (float)(BY_PIECE ? others : N - all);
    some = all > 0;
    if constexpr (LAYOUT != FULL) {
#pragma unroll
      for (int i = 0; i < WORDS; ++i)
        keep[i] = LAYOUT == APART || sizeof(T) == 4 ? (in(i, C) ? 0xffffffffu : 0u)
                                                    : (in(2 * i, C) ? 0xffffu : 0u) | (in(2 * i + 1, C) ? 0xffff0000u : 0u);
    }
  }
  __device__ __forceinline__ int at(int j) const { return first[j / V] + j % V; }
  __device__ __forceinline__ bool in(int j, int C) const { return LAYOUT == FULL || (at(j) >= 0 && at(j) < C); }
  __device__ __forceinline__ bool whole(int k) const { return LAYOUT == FULL || count[k] == V; }
  __device__ __forceinline__ bool any(int k) const { return LAYOUT == FULL || count[k] > 0; }

  // zeros for the values that are not the row's
  __device__ __forceinline__ void clear(float2* v) const {
#pragma unroll
    for (int i = 0; i < N / 2; ++i)
      v[i] = make_float2(__uint_as_float(__float_as_uint(v[i].x) & keep[2 * i]), __uint_as_float(__float_as_uint(v[i].y) & keep[2 * i + 1]));
  }

  __device__ __forceinline__ void param(const void* p, int f32, float missing, int C, float2* v) const {
    float t[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      t[j] = 0.f;
      if (in(j, C))
        t[j] = !p ? missing
                  : (f32 ? load_in(static_cast<const float*>(p) + at(j)) : to_f32(load_in(static_cast<const bf16*>(p) + at(j))));
    }
#pragma unroll
    for (int i = 0; i < N / 2; ++i) v[i] = make_float2(t[2 * i], t[2 * i + 1]);
  }
};

// the first m, or with `last` the last m, values of a 16-byte piece at dst, 0 < m < 16 / SIZE: a store for each power of
// two in m, each aligned to its size
template <int SIZE>
__device__ __forceinline__ void store_some(char* dst, uint4 piece, int m, bool last) {
  const uint32_t w[4] = {piece.x, piece.y, piece.z, piece.w};
  const int bytes = m * SIZE;
  char* at = last ? dst + 16 - bytes : dst;
  // from the piece's end inwards, or from its start
  if (bytes & 8) *reinterpret_cast<uint2*>(last ? dst + 8 : dst) = last ? make_uint2(w[2], w[3]) : make_uint2(w[0], w[1]);
  const bool far = bytes & 8;
  if (bytes & 4)
    *reinterpret_cast<uint32_t*>(last ? dst + (far ? 4 : 12) : dst + (far ? 8 : 0)) = last ? (far ? w[1] : w[3]) : (far ? w[2] : w[0]);
  if constexpr (SIZE == 2)
    if (bytes & 2) {
      // word of the odd value: the one that holds the first (last) value kept
      const int i = last ? (16 - bytes) / 4 : (bytes - 2) / 4;
      const uint32_t u = i == 0 ? w[0] : (i == 1 ? w[1] : (i == 2 ? w[2] : w[3]));
      *reinterpret_cast<uint16_t*>(last ? at : dst + bytes - 2) = (uint16_t)(last ? u >> 16 : u);
    }
}

// A lane's part of a row as it lies in memory.
template <typename T, Layout LAYOUT, int N>
struct Part {
  using At = Lane<T, LAYOUT, N>;
  static constexpr int V = At::V, K = At::K;
  Raw<T, V> raw[K];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int k = 0; k < K; ++k) raw[k].zero();
  }
  // (what is not of the row stays as it was, or is a neighbour's); inner: no first or last row, whose pieces could
  // reach out of the tensor
  __device__ __forceinline__ void load(const At& at, const T* row, bool inner) {
    if (LAYOUT != PIECES || inner) {
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (at.any(k)) raw[k].load(row + at.first[k]);
    } else {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const T* const src = row + at.first[k];
        alignas(16) T t[V];
        const int from = at.first[k] < 0 ? V - at.count[k] : 0;
#pragma unroll
        for (int i = 0; i < V; ++i) t[i] = i >= from && i < from + at.count[k] ? load_in(src + i) : from_f32<T>(0.f);
        if constexpr (LAYOUT == PIECES) raw[k].piece = *reinterpret_cast<const uint4*>(t);
      }
    }
  }
  // the lane's values, and `fill` for those that are not the row's
  __device__ __forceinline__ void values(const At& at, float fill, float2* v) const {
    float t[N];
    uint32_t f = __float_as_uint(fill);
    if (LAYOUT == PIECES && sizeof(T) == 2) f = __byte_perm(f, f, 0x3232);  // (a value of the row, or 0: exact in 16 bits)
#pragma unroll
    for (int k = 0; k < K; ++k) {
      Raw<T, V> r = raw[k];
      if constexpr (LAYOUT == PIECES) {
        uint32_t w[4] = {r.piece.x, r.piece.y, r.piece.z, r.piece.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = (w[i] & at.keep[4 * k + i]) | (f & ~at.keep[4 * k + i]);
        r.piece = make_uint4(w[0], w[1], w[2], w[3]);
      }
      r.values(t + k * V);
      if constexpr (LAYOUT == APART)
        t[k] = __uint_as_float((__float_as_uint(t[k]) & at.keep[k]) | (f & ~at.keep[k]));
    }
#pragma unroll
    for (int i = 0; i < N / 2; ++i) v[i] = make_float2(t[2 * i], t[2 * i + 1]);
  }
  // A value of the row from its L lanes (PIECES: the second piece is the row's whatever the first one holds).
  template <int L>
  __device__ __forceinline__ float lead() const {
    uint32_t w;
    if constexpr (LAYOUT == APART)
      w = __float_as_uint(to_f32(raw[0].one[0]));
    else
      w = raw[0].piece.x;
    w = __shfl_sync(0xffffffffu, w, LAYOUT == PIECES ? 1 : 0, L);
    return __uint_as_float(LAYOUT != APART && sizeof(T) == 2 ? w << 16 : w);
  }
  // piece k as it goes to memory
  static __device__ __forceinline__ uint4 words(const float2* v, int k) {
    if constexpr (sizeof(T) == 4) {
      return make_uint4(__float_as_uint(v[2 * k].x), __float_as_uint(v[2 * k].y), __float_as_uint(v[2 * k + 1].x),
                        __float_as_uint(v[2 * k + 1].y));
    } else {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 h = __float22bfloat162_rn(v[4 * k + i]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
      return make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  static __device__ __forceinline__ void store(const At& at, T* row, const float2* v) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      T* const dst = row + at.first[k];
      if constexpr (LAYOUT == APART) {
        if (at.any(k)) *dst = from_f32<T>(k & 1 ? v[k / 2].y : v[k / 2].x);
      } else {
        const uint4 w = words(v, k);
        if (at.whole(k))
          *reinterpret_cast<uint4*>(dst) = w;
        else if (at.any(k))
          store_some<sizeof(T)>(reinterpret_cast<char*>(dst), w, at.count[k], k == 0 && at.first[k] < 0);
      }
    }
  }
};

// values between the 16-byte address before row r and the row
template <typename T>
__device__ __forceinline__ int row_head(const void* x, int64_t stride, int64_t r) {
  return (int)((reinterpret_cast<uintptr_t>(static_cast<const T*>(x) + r * stride) & 15) / sizeof(T));
}

// Stores of rows of L lanes that start anywhere.  A row's first and last piece, where it is not the row's alone, goes
// through shared memory (two slots for each of the warp's rows), from where every lane takes single words whose place
// in the rows does not change from step to step: 14 instructions where stores of what each lane has of a piece, in all
// the sizes it can have, take a hundred.
template <typename T, Layout LAYOUT, int N, int L>
struct Edges {  // (of the other layouts: none)
  template <typename... A>
  __device__ __forceinline__ explicit Edges(const A&...) {}
};
template <typename T, int N, int L>
struct Edges<T, PIECES, N, L> {
  using At = Lane<T, PIECES, N>;
  static constexpr int V = At::V, K = At::K, ROWS = 32 / L, SLOTS = 2 * ROWS, PER = (4 * SLOTS + 31) / 32;
  static constexpr int OF_WORD = 4 / sizeof(T);
  uint4* slots;      // of the warp
  bool start, end[K];  // whether this lane's first piece starts the row in part, a piece ends it in part
  int slot;          // of the row's start; its end's is the next
  T* to[PER];
  uint32_t row[PER];  // of a word, among the warp's next rows
  uint32_t on;        // bits: the values of the words that are stored
  // r: this lane's row
  __device__ __forceinline__ Edges(const At& at, const LayerNorm& p, uint4* shared, uint32_t r, T* y) {
    const int lane = threadIdx.x & 31, sub = lane / L;
    slots = shared + (threadIdx.x >> 5) * SLOTS;
    slot = 2 * sub;
    start = at.first[0] < 0 && lane % L == 0;
#pragma unroll
    for (int k = 0; k < K; ++k) end[k] = !at.whole(k) && at.any(k) && !(k == 0 && start);
    on = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int word = lane + 32 * i, s = word / 4;
      const uint32_t first = r - sub, which = s / 2;
      row[i] = first + which;
      const int head = row_head<T>(p.x, p.xs, row[i]), last = (p.C + head - 1) / V;  // (its last piece)
      const int c = (s & 1 ? last * V : 0) - head + word % 4 * OF_WORD;
      to[i] = y + ((int64_t)row[i] - r) * p.ys + c;
#pragma unroll
      for (int e = 0; e < OF_WORD; ++e) {
        const bool part = s & 1 ? (p.C + head) % V != 0 && c + e < p.C : head > 0 && c + e >= 0;
        if (s < SLOTS && part) on |= 1u << (i * OF_WORD + e);
      }
    }
  }
  __device__ __forceinline__ void store(const At& at, T* y, const float2* v, bool in, uint32_t n) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const uint4 w = Part<T, PIECES, N>::words(v, k);
      if (in && at.whole(k)) *reinterpret_cast<uint4*>(y + at.first[k]) = w;
      if (k == 0 && start) slots[slot] = w;
      if (end[k]) slots[slot + 1] = w;
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const uint32_t w = reinterpret_cast<const uint32_t*>(slots)[(threadIdx.x & 31) + 32 * i < 4 * SLOTS ? (threadIdx.x & 31) + 32 * i : 0];
      if (row[i] < n) {
        if constexpr (sizeof(T) == 4) {
          if (on >> i & 1) *reinterpret_cast<uint32_t*>(to[i]) = w;
        } else {
          if (on >> (2 * i) & 1) *reinterpret_cast<uint16_t*>(to[i]) = (uint16_t)w;
          if (on >> (2 * i + 1) & 1) *reinterpret_cast<uint16_t*>(to[i] + 1) = (uint16_t)(w >> 16);
        }
      }
    }
    __syncwarp();
  }
  __device__ __forceinline__ void step(uint32_t rows, int64_t values) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      row[i] += rows;
      to[i] += values;
    }
  }
};

// ---- sums over the L neighbouring lanes of a row, or over all threads of a CTA
template <int L>
struct LaneSum {
  __device__ __forceinline__ float operator()(float a) const {
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
    return a;
  }
  __device__ __forceinline__ float2 operator()(float2 a) const { return make_float2((*this)(a.x), (*this)(a.y)); }
};
template <int WARPS>
struct CtaSum {
  static constexpr int FLOATS = 4 * WARPS;
  static_assert(WARPS % 4 == 0, "each of the buffers starts at 16 bytes");
  // Two of WARPS for single sums, in turn, and one for pairs: a thread writes to one of them again only behind another
  // barrier, which all pass when they have read it (pairs are never summed twice without single sums between).
  float* buffer;
  int at = 0;
  // (zeros for the warps that the CTA has not)
  __device__ __forceinline__ explicit CtaSum(float* b) : buffer(b) {
    for (int k = threadIdx.x; k < FLOATS; k += blockDim.x) b[k] = 0.f;
    __syncthreads();
  }
  __device__ __forceinline__ float2 operator()(float2 a) {
    a = LaneSum<32>()(a);
    float2* const b = reinterpret_cast<float2*>(buffer + 2 * WARPS);
    if ((threadIdx.x & 31) == 0) b[threadIdx.x >> 5] = a;
    __syncthreads();
    const float4 t = total(reinterpret_cast<const float*>(b), 2 * WARPS);
    return make_float2(t.x + t.z, t.y + t.w);
  }
  __device__ __forceinline__ float operator()(float a) {
    a = LaneSum<32>()(a);
    float* const b = buffer + at;
    at ^= WARPS;
    if ((threadIdx.x & 31) == 0) b[threadIdx.x >> 5] = a;
    __syncthreads();
    const float4 t = total(b, WARPS);
    return (t.x + t.y) + (t.z + t.w);
  }
  static __device__ __forceinline__ float4 total(const float* b, int floats) {
    float4 t = *reinterpret_cast<const float4*>(b);
#pragma unroll
    for (int k = 4; k < floats; k += 4) {
      const float4 u = *reinterpret_cast<const float4*>(b + k);
      t.x += u.x, t.y += u.y, t.z += u.z, t.w += u.w;
    }
    return t;
  }
};

template <int H>
__device__ __forceinline__ float2 tree(float2* v) {  // (v is used up)
#pragma unroll
  for (int o = H / 2; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < o; ++i) v[i] = add2(v[i], v[i + o]);
  return v[0];
}
// A row's values become xhat; rstd is returned.  lead: one of the row's values, which those that are not the row's hold
// too.  Sums are taken of x - lead: a row of equal values comes out as zeros, an offset common to the row costs no
// accuracy, and lead is never further from the mean than sqrt(C) standard deviations: a row in which it is alone in size
// loses that many units in the last place, others a few.
//   The values that are not the row's are then -mean.  fp32 rows leave out the squares of pieces that have none of the
// row's values; of the pieces at a row's ends, and in 16 bits of all, they are taken off their lane's sum, with an error of
// a unit in the last place of mean^2 for each.  (The row's own sum holds mean^2 once, for lead: all that are off in a lane of
// a one-hot row of 4097 would make rstd wrong by 6e-5, below 16 bits' 2^-9.)
template <typename T, Layout LAYOUT, int N, typename Sum>
__device__ __forceinline__ float normalise(const Lane<T, LAYOUT, N>& at, float2* v, float lead, const LayerNorm& p, Sum& sum) {
  using At = Lane<T, LAYOUT, N>;
  constexpr int H = N / 2;
  float2 a[H];
#pragma unroll
  for (int i = 0; i < H; ++i) a[i] = v[i] = add2(v[i], both(-lead));
  const float2 s = tree<H>(a);
  const float mean = sum(s.x + s.y) * p.inv_C;
#pragma unroll
  for (int i = 0; i < H; ++i) v[i] = add2(v[i], both(-mean));
  float q = 0.f;
  if constexpr (At::BY_PIECE) {
    constexpr int P = At::V / 2;
#pragma unroll
    for (int k = 0; k < At::K; ++k) {
      float2 qk = mul2(v[k * P], v[k * P]);
#pragma unroll
      for (int i = 1; i < P; ++i) qk = fma2(v[k * P + i], v[k * P + i], qk);
      q = fmaf(qk.x + qk.y, at.has[k], q);
    }
  } else {
    if constexpr (LAYOUT == APART && sizeof(T) == 4) at.clear(v);
    float2 q0 = mul2(v[0], v[0]), q1 = mul2(v[1], v[1]);
#pragma unroll
    for (int i = 2; i < H; i += 2) {
      q0 = fma2(v[i], v[i], q0);
      q1 = fma2(v[i + 1], v[i + 1], q1);
    }
    const float2 qq = add2(q0, q1);
    q = qq.x + qq.y;
  }
  if (At::BY_PIECE)
    q = fmaf(-at.off * mean, mean, q);
  else if (LAYOUT == PIECES || (LAYOUT == APART && sizeof(T) == 2))
    q = at.some ? fmaf(-at.off * mean, mean, q) : 0.f;
  // (a lane's share of the variance: values of up to 1e18, whose 2e18 of deviation 16 values of a lane square to less than
  // 2^128, in rows of any width)
  const float rstd = rsqrtf(sum(q * p.inv_C) + p.eps);
#pragma unroll
  for (int i = 0; i < H; ++i) v[i] = mul2(v[i], both(rstd));
  return rstd;
}

__device__ __forceinline__ float reciprocal(float a) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(a));
  return r;
}

// s = 1 / (1 + exp(-z)).  Both functions are the hardware's (exp2 within 2 units in the last place of an argument that
// rounds by |z| units, which count where exp(-z) outweighs the 1; the reciprocal within 1), and two values share a
// reciprocal of their product: 12 of them instead of 16 for 8 values, whose pipe bounds 16-bit rows.  Values
// whose product could overflow, or that are not numbers, are taken one by one.  There fp32 rows take exp(z) itself where
// the 1 is lost beside exp(-z): s below 2^-126, whose z s is still a normal number, comes out as a subnormal one.  (In 16
// bits z s is zero from 1e-36 down: the same made gradients of 300 007 rows of 97 4 % slower, of 8192 channels 7 %.)
__device__ __forceinline__ float sigmoid(float z, float a) {  // a: 1 + exp(-z)
  float r;
  asm("ex2.approx.f32 %0, %1;" : "=f"(r) : "f"(z * 1.44269504f));
  return a > 0x1p62f ? r : reciprocal(a);
}
template <typename T, int H>
__device__ __forceinline__ void sigmoid(const float2* z, float2* s) {  // of 2 H values
  float2 a[H], t[H];
#pragma unroll
  for (int i = 0; i < H; ++i) {
    const float2 e = mul2(z[i], both(-1.44269504f));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(a[i].x) : "f"(e.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(a[i].y) : "f"(e.y));
    t[i] = a[i] = add2(a[i], both(1.f));
  }
  const float2 top = tree<H>(t);
  if (top.x + top.y <= 0x1p62f) {
#pragma unroll
    for (int i = 0; i < H; ++i) s[i] = mul2(both(reciprocal(a[i].x * a[i].y)), make_float2(a[i].y, a[i].x));
  } else {
#pragma unroll
    for (int i = 0; i < H; ++i)
      s[i] = sizeof(T) == 4 ? make_float2(sigmoid(z[i].x, a[i].x), sigmoid(z[i].y, a[i].y))
                            : make_float2(reciprocal(a[i].x), reciprocal(a[i].y));
  }
}

// lanes of a row: N channels each (`head`: and the values before its start); a power of two up to a warp, then whole
// warps
inline int row_lanes(int N, int C, int head) {
  const int need = (C + head + N - 1) / N;
  if (need > 32) return (need + 31) / 32 * 32;
  int l = 2;
  while (l < need) l *= 2;
  return l;
}

// (volatile: not kept in registers over a loop)
__device__ __forceinline__ float4 load_shared(const float4* a) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"((uint32_t)__cvta_generic_to_shared(a))
               : "memory");
  return v;
}

// A lane's weights and biases: in registers, or in shared memory of its own (16 bytes of every lane side by side).
template <int N, bool SHARED>
struct Params {
  float2 w_[SHARED ? 1 : N / 2], b_[SHARED ? 1 : N / 2];
  float4* at_;
  int lanes_;
  static constexpr int BYTES = 2 * N * 4;  // of a lane
  template <typename At>
  __device__ __forceinline__ Params(const At& at, const LayerNorm& p, void* shared, int lane, int lanes)
      : at_(static_cast<float4*>(shared) + lane), lanes_(lanes) {
    if constexpr (SHARED) {
      float2 t[N / 2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        at.param(h ? p.b : p.w, p.param_f32, h ? 0.f : 1.f, p.C, t);
#pragma unroll
        for (int i = 0; i < N / 4; ++i)
          at_[(h * (N / 4) + i) * lanes] = make_float4(t[2 * i].x, t[2 * i].y, t[2 * i + 1].x, t[2 * i + 1].y);
      }
    } else {
      at.param(p.w, p.param_f32, 1.f, p.C, w_);
      at.param(p.b, p.param_f32, 0.f, p.C, b_);
    }
  }
  // of values 8 c .. 8 c + 7
  __device__ __forceinline__ void get(int h, int c, float2* v) const {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if constexpr (SHARED) {
        const float4 t = load_shared(at_ + (h * (N / 4) + 2 * c + i) * lanes_);
        v[2 * i] = make_float2(t.x, t.y), v[2 * i + 1] = make_float2(t.z, t.w);
      } else {
        v[2 * i] = (h ? b_ : w_)[4 * c + 2 * i], v[2 * i + 1] = (h ? b_ : w_)[4 * c + 2 * i + 1];
      }
    }
  }
  __device__ __forceinline__ void weight(int c, float2* v) const { get(0, c, v); }
  __device__ __forceinline__ void bias(int c, float2* v) const { get(1, c, v); }
};

// A lane's sums of the parameters' gradients, kept the same way.
template <int N, bool SHARED>
struct Sums {
  float2 v_[2][SHARED ? 1 : N / 2];
  float4* at_;
  int lanes_;
  static constexpr int BYTES = 2 * N * 4;  // of a lane
  __device__ __forceinline__ Sums(void* shared, int lane, int lanes) : at_(static_cast<float4*>(shared) + lane), lanes_(lanes) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      if constexpr (SHARED)
        at_[i * lanes] = make_float4(0.f, 0.f, 0.f, 0.f);
      else
        v_[0][i] = v_[1][i] = both(0.f);
    }
  }
  // values 8 c .. 8 c + 7 of g xhat and of g
  __device__ __forceinline__ void add(int c, const float2* g, const float2* xhat) {
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      if constexpr (SHARED) {
        float4 *const w = at_ + (2 * c + i / 2) * lanes_, *const b = w + (N / 4) * lanes_;
        float4 t = *w, u = *b;
        const float2 t0 = fma2(g[i], xhat[i], make_float2(t.x, t.y)), t1 = fma2(g[i + 1], xhat[i + 1], make_float2(t.z, t.w));
        const float2 u0 = add2(g[i], make_float2(u.x, u.y)), u1 = add2(g[i + 1], make_float2(u.z, u.w));
        *w = make_float4(t0.x, t0.y, t1.x, t1.y);
        *b = make_float4(u0.x, u0.y, u1.x, u1.y);
      } else {
#pragma unroll
        for (int k = i; k < i + 2; ++k) {
          v_[0][4 * c + k] = fma2(g[k], xhat[k], v_[0][4 * c + k]);
          v_[1][4 * c + k] = add2(g[k], v_[1][4 * c + k]);
        }
      }
    }
  }
  // the sums of g xhat (which: 0) and g (1), value j
  __device__ __forceinline__ float get(int which, int j) const {
    if constexpr (SHARED) {
      const float4 t = at_[(which * (N / 4) + j / 4) * lanes_];
      return j % 4 == 0 ? t.x : (j % 4 == 1 ? t.y : (j % 4 == 2 ? t.z : t.w));
    } else {
      return j & 1 ? v_[which][j / 2].y : v_[which][j / 2].x;
    }
  }
};

struct RowPlan {
  Layout layout;
  int values, lanes;  // of a lane, of a row
};
struct Operand {
  const void* at;  // null: none
  int64_t stride;
};

// Values of a lane.  Rows of up to 32 lanes: two pieces, so that 32 bytes of each row are in flight for a lane and the
// row's sums take few steps; but one piece of 16 bits in the backward where a row starts anywhere (300 007 rows of 97
// 75 us; with two, whose masks leave too few registers, 87), and 8 single values.  Four pieces of fp32 where a row then
// still fits a warp, and where it takes a CTA (gradients of 20 011 rows of 2048 87 us, 99 with two).
constexpr int LN_WIDE = 16, LN_APART = 8;
template <typename T, bool GRAD>
constexpr int narrow_values(Layout layout) {
  return sizeof(T) == 4 || layout == APART || (GRAD && layout == PIECES) ? 8 : 16;
}

// lanes of more than a warp
constexpr bool may_be_wide(Layout layout, int values) { return layout == APART || values == LN_WIDE; }

template <typename T, bool GRAD>
RowPlan row_plan(int64_t n, int C, std::initializer_list<Operand> operands) {
  constexpr int V = 16 / sizeof(T);
  bool alike = true, start = true, apart = true;
  const Operand& x = *operands.begin();
  for (const Operand& o : operands) {
    if (!o.at) continue;
    alike = alike && ((reinterpret_cast<uintptr_t>(o.at) - reinterpret_cast<uintptr_t>(x.at)) & 15) == 0 &&
            (o.stride - x.stride) % V == 0;
    start = start && (reinterpret_cast<uintptr_t>(o.at) & 15) == 0 && o.stride % V == 0;
    apart = apart && (o.stride > 0 || n <= 1);
  }
  const int head = start ? 0 : V - 1;
  auto plan = [&](Layout layout) {
    int values = narrow_values<T, GRAD>(layout);
    if (row_lanes(values, C, head) > 32) values = LN_WIDE;
    return RowPlan{layout, values, row_lanes(values, C, head)};
  };
  const RowPlan full = plan(FULL), pieces = plan(PIECES);
  if (start && full.lanes * full.values == C) return full;
  // (rows that repeat: a neighbour's values need not lie inside the tensor)
  const bool any = alike && apart && C > V && pieces.lanes * pieces.values <= MACE_LAYER_NORM_MAX_CHANNELS;
  return any ? pieces : RowPlan{APART, LN_APART, row_lanes(LN_APART, C, 0)};
}

inline uint32_t inner_rows(int64_t n) { return n > 2 * LN_TURN ? (uint32_t)(n - 2 * LN_TURN) : 0; }

inline bool bad_rows(int32_t dtype, int32_t param_dtype, int64_t n, int32_t C, float eps, int32_t activation) {
  return (dtype != MACE_F32 && dtype != MACE_BF16) || (param_dtype != MACE_F32 && param_dtype != MACE_BF16) || n < 0 ||
         n > INT32_MAX || C < 1 || C > MACE_LAYER_NORM_MAX_CHANNELS || !(eps >= 0.f) || !std::isfinite(eps) ||
         (activation != MACE_ACT_NONE && activation != MACE_ACT_SILU);
}

// Whether n rows of C values that are written meet what is read: n rows as well, or `one` of C values.  Rows of two
// strides lie apart where no multiple of the strides' common divisor brings one to the other: exact for equal strides
// (slots of one table) and for one row; interleaved rows of unlike strides count as meeting unless that shows them apart.
struct Span {
  const void* at;  // null: none
  int64_t stride;  // in values
  int size;        // of a value
  bool one;
};
inline bool rows_meet(const Span& out, const Span& in, int64_t n, int C) {
  if (!out.at || !in.at || n < 1) return false;
  const int64_t row_out = (int64_t)C * out.size, row_in = (int64_t)C * in.size;
  const int64_t step_out = n > 1 ? out.stride * out.size : 0, step_in = n > 1 && !in.one ? in.stride * in.size : 0;
  const uintptr_t o = reinterpret_cast<uintptr_t>(out.at), i = reinterpret_cast<uintptr_t>(in.at);
  if (o + (n - 1) * step_out + row_out <= i || i + (n - 1) * step_in + row_in <= o) return false;
  const int64_t period = std::gcd(step_out, step_in);
  if (period == 0) return true;
  const int64_t d = (int64_t)(i - o) % period, behind = d < 0 ? d + period : d;  // of a row that is read behind one that is written
  return behind < row_out || period - behind < row_in;
}

// f(layout, values) of a plan as constants
template <typename T, bool GRAD, typename F>
int with_plan(const RowPlan& plan, F&& f) {
  auto go = [&](auto layout) {
    constexpr int narrow = narrow_values<T, GRAD>(decltype(layout)::value);
    if constexpr (decltype(layout)::value != APART && narrow != LN_WIDE)
      if (plan.values == LN_WIDE) return f(layout, std::integral_constant<int, LN_WIDE>{});
    return f(layout, std::integral_constant<int, narrow>{});
  };
  switch (plan.layout) {
    case FULL: return go(std::integral_constant<Layout, FULL>{});
    case PIECES: return go(std::integral_constant<Layout, PIECES>{});
    default: return go(std::integral_constant<Layout, APART>{});
  }
}

// f(lanes) of a row of up to 32 lanes; one whose lanes have more values than narrow ones has a whole warp
template <bool WARP, typename F>
int with_lanes(int lanes, F&& f) {
  if constexpr (!WARP) {
    switch (lanes) {
      case 2: return f(std::integral_constant<int, 2>{});
      case 4: return f(std::integral_constant<int, 4>{});
      case 8: return f(std::integral_constant<int, 8>{});
      case 16: return f(std::integral_constant<int, 16>{});
      default: break;
    }
  }
  return f(std::integral_constant<int, 32>{});
}

}  // namespace mace
