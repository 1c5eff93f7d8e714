// Species-indexed linear map (reference tensor_product.py:1046-1305 with a
// one-hot second input) on rows grouped by species, and its weight gradient,
// on the 5th-generation tensor cores:
//   y[r]  = alpha x[r] W[g(r)]                    (128 grouped rows x NT columns per tile, K = channels)
//   dW[g] = alpha sum over r in g of x[r]^T dy[r]  (128 input channels x NT columns per tile, K = rows)
//
// Arithmetic.  An fp32 operand is split into three bf16 pieces x = h + m + l
// (8 bits each: the 24 bits of x exactly) and six of the nine products are
// kept (h h, h m, m h, m m, h l, l h; the dropped ones are below 2^-21 of
// x w, 2^-24 on average), all kind::f16 MMAs: the instruction count of a 3xTF32 split
// with 3/4 of its operand bytes.  bf16 data is one piece; 8-bit checkpoint
// values are exact in one bf16 piece and their row scale is folded into dy.
// The tensor core truncates when it accumulates, so an accumulator takes one
// 64-wide step of K, smallest products first, and the epilogue warps add the
// steps in fp32 registers (bf16 alone, whose result is rounded to 8 bits, takes
// several steps).
//
// Roles of a CTA of the map (16 warps, one CTA per SM, a share of the tiles of equal cost):
//   warps 0-3   operand A: own 32 TMEM lanes each, fetch their rows with 16-byte
//               cp.async through a private ring (gathered by `order`), split
//               them in registers and store them to TMEM
//   warps 4-7   operand B: the weights into 128B-swizzled K-major shared-memory
//               images, kept while the tiles share them; warp 4 issues the MMAs
//               (a 17th warp would cut every thread to 96 registers)
//   warps 8-15  epilogue: TMEM -> fp32 registers -> memory
// handing over through mbarriers only.  600 000 fp32 rows 128 -> 128 take 124 us
// (5.0 TB/s; 94 is what HBM needs): no role is busy all the time, the hand-over
// between them is what is left.  A tile's 128 rows by NT columns are what TMEM
// holds twice beside two stages of A; K goes in steps of 64, what an
// accumulator may take.  Every wait is bounded (about 2 s): one
// that gives up raises the CTA's abort flag, which ends every other wait, and
// TC_ERR_TIMEOUT in g_species_error.  species_wgrad.cuh has the weight
// gradient, species_direct.cuh both for bf16 rows that need no conversion.
//
// Rows may start at any alignment: a segment is fetched as the 16-byte units
// that contain it (its end clipped by the copy's source size) and shifted when
// it is read from shared memory (template VEC = 0; VEC = 1 when every row is
// 16-byte aligned).
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "species.cuh"
#include "tc.cuh"

namespace mace {

namespace {

constexpr int SL_THREADS = 16 * 32;
constexpr int SL_KC = 64;              // K of one accumulation step
constexpr int SL_IMG = 128 * 128;      // bytes of one piece of a B image of up to 128 rows of 64 bf16
constexpr int SL_LONG = 8;             // weight gradient of bf16: steps accumulated in TMEM
constexpr int SL_STEPS = 2048;         // weight gradient: steps that a share may add into one fp32 sum
constexpr int SL_D = 0;                // TMEM columns: two accumulators of 128
constexpr int SL_A = 256;              // then two A stages
constexpr uint32_t SL_TMEM = 512;

__device__ int g_species_error;  // TC_ERR_TIMEOUT once a bounded wait gave up

// feature rows: element (node, m, c) at data + node * node_stride + m * comp_stride + c
struct RowView {
  const char* data;
  int64_t sn, sm;       // bytes
  int width;            // channels
  uint32_t sn16, sm16;  // aligned rows: 16 bytes
};

struct SlParams {
  RowView a;            // map: x; weight gradient: x or its 8-bit checkpoint
  RowView b;            // weight gradient: dy
  const float* a_scale; // 8-bit checkpoint scales (n, d, ka_blocks)
  int ka_blocks;
  const void* w;        // map: weights (G, K, N), or (G, N, K) when transposed
  int transposed;
  void* out;            // map: y; weight gradient: dW (G, K, N)
  int64_t out_sn, out_sm;     // map: elements
  uint32_t out_n32, out_m32;  // map: the same in 16 bytes (vst) or, where all offsets fit 32 bits (out32), elements
  int out32;
  int vst;              // map: rows of `out` are whole 16-byte pieces; weight gradient: bytes of a vector store (32, 16, 0)
  float* part;          // weight gradient: partial tiles
  int* spans;           // weight gradient: a group's first share, bit 15 if it begins inside it, and its last in the
                        // upper 16 bits (-1: no rows), written by CTA 0 for the join
  const int32_t* order;
  const int32_t* offsets;
  int64_t n;
  int d, G;
  uint32_t div_mul, div_shift;  // x / d for x < 2^31, d > 1: the high word of x div_mul, shifted
  int K, N;             // map: K summed channels, N outputs; weight gradient: K x N of dW
  int w_vec;            // map: rows of the weights are 16-byte aligned
  int NT;               // tile columns: 32, 64, 96 or 128
  int start;            // map: what the weight images of a group cost, in half row tiles
  int img, slots;       // map: bytes of one piece of a weight image, slots for the images of a step
  int n_ct, n_kt;       // column tiles; weight gradient: row (channel) tiles
  int shares;           // weight gradient: CTAs along the rows
  float alpha;
};

// ------------------------------------------------------------------ helpers
__device__ __forceinline__ constexpr uint32_t idesc_bf16(int N) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | ((128u >> 4) << 24);
}

// D[tmem] (+)= A[tmem] . B[smem]^T in bf16: A's M rows are the TMEM lanes, two
// consecutive K elements per 32-bit column; B's descriptor as its two halves
__device__ __forceinline__ void mma_bf16_ta(uint32_t d, uint32_t a, uint32_t blo, uint32_t bhi, uint32_t idesc,
                                            bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 b, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, {%6, %6, %6, %6}, p;\n\t}" ::"r"(d),
      "r"(a), "r"(blo), "r"(bhi), "r"(idesc), "r"((uint32_t)acc), "r"(0u)
      : "memory");
}

__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t phase, uint32_t suspend_ns) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(phase), "r"(suspend_ns)
      : "memory");
  return ok != 0;
}

// Bounded wait for a phase; false once the CTA's abort flag is up (a wait that gives up raises it).  A phase that
// is complete costs one try: reading the abort flag and the global timer before it would cost more than the hand-over.
__device__ __forceinline__ bool wait_phase(uint32_t bar, uint32_t phase, volatile int* abort) {
  if (mbar_try(bar, phase, 0)) return true;
  return tc::mbar_wait_or_abort(bar, phase, abort);
}

// One arrival for what the lanes of a warp have done (each behind its own fence where another proxy reads it).  An
// arrival by every thread queues on the barrier.
__device__ __forceinline__ void warp_arrive(uint32_t bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) tc::mbar_arrive(bar);
}

// true on one lane of a converged warp; the compiler knows the branch is uniform
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r != 0;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// 16 bytes, or zeros
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void* src, bool zero) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %2, 0;\n\t"
      "cp.async.cg.shared.global [%0], [%1], 16, p;\n\t}" ::"r"(dst),
      "l"(src), "r"((uint32_t)zero)
      : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Shared memory through pointers, so that constant offsets become part of the instruction
template <typename T>
__device__ __forceinline__ T load_as(const uint8_t* a) { return *reinterpret_cast<const T*>(a); }
template <typename T>
__device__ __forceinline__ float load_f32(const uint8_t* a) { return to_f32(load_as<T>(a)); }
__device__ __forceinline__ void store_piece(uint8_t* a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  *reinterpret_cast<uint4*>(a) = make_uint4(x, y, z, w);
}
// eight consecutive values
__device__ __forceinline__ void load_eight(const uint8_t* a, float* v, float) {
  const uint4 x = load_as<uint4>(a), y = load_as<uint4>(a + 16);
  const uint32_t w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = __uint_as_float(w[k]);
}
__device__ __forceinline__ void load_eight(const uint8_t* a, float* v, bf16) {
  const uint4 x = load_as<uint4>(a);
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    v[2 * k] = __uint_as_float(w[k] << 16);
    v[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
  }
}

// two values rounded to bf16, x0 in the low half
__device__ __forceinline__ uint32_t pack_bf16(float x0, float x1) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(x1), "f"(x0));
  return r;
}

// (x0 - y0, x1 - y1)
__device__ __forceinline__ void sub2(float& x0, float& x1, uint32_t y0, uint32_t y1) {
  asm("{\n\t.reg .b64 a, b;\n\t"
      "mov.b64 a, {%0, %1};\n\t"
      "mov.b64 b, {%2, %3};\n\t"
      "sub.rn.f32x2 a, a, b;\n\t"
      "mov.b64 {%0, %1}, a;\n\t}"
      : "+f"(x0), "+f"(x1)
      : "r"(y0), "r"(y1));
}

__device__ __forceinline__ void add2(float& x0, float& x1, uint32_t y0, uint32_t y1) {
  asm("{\n\t.reg .b64 a, b;\n\t"
      "mov.b64 a, {%0, %1};\n\t"
      "mov.b64 b, {%2, %3};\n\t"
      "add.rn.f32x2 a, a, b;\n\t"
      "mov.b64 {%0, %1}, a;\n\t}"
      : "+f"(x0), "+f"(x1)
      : "r"(y0), "r"(y1));
}

// (x0 + z y0, x1 + z y1)
__device__ __forceinline__ void fma2(float& x0, float& x1, uint32_t y0, uint32_t y1, float z) {
  asm("{\n\t.reg .b64 a, b, c;\n\t"
      "mov.b64 a, {%0, %1};\n\t"
      "mov.b64 b, {%2, %3};\n\t"
      "mov.b64 c, {%4, %4};\n\t"
      "fma.rn.f32x2 a, b, c, a;\n\t"
      "mov.b64 {%0, %1}, a;\n\t}"
      : "+f"(x0), "+f"(x1)
      : "r"(y0), "r"(y1), "f"(z));
}

// the bf16 pieces of two values, packed: P = 3: x = h + m + l, each the leading
// 8 bits of what is left (exact, and no finite value becomes infinite);
// P = 1: x rounded (exact where it is used)
template <int P>
__device__ __forceinline__ void split2(float x0, float x1, uint32_t* out) {
  if constexpr (P == 1) {
    out[0] = pack_bf16(x0, x1);
  } else {
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      const uint32_t u0 = __float_as_uint(x0), u1 = __float_as_uint(x1);
      out[k] = __byte_perm(u0, u1, 0x7632);
      // (the first value's piece back by a multiplication: masks and permutes share one pipe, half as wide)
      if (k < 2) sub2(x0, x1, out[k] * 65536u, u1 & 0xffff0000u);
    }
  }
}

__device__ __forceinline__ void tmem_st16u(uint32_t a, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(a),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}

__device__ __forceinline__ void tmem_ld16u(uint32_t a, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(a)
      : "memory");
}

// 16 consecutive values of a result row, `left` of them inside it
template <typename T>
__device__ __forceinline__ void store16(T* dst, const float* v, int left, int vst) {
  uint32_t w[16];
  constexpr int W = 16 * sizeof(T) / 4;
#pragma unroll
  for (int k = 0; k < W; ++k) {
    if constexpr (sizeof(T) == 4)
      w[k] = __float_as_uint(v[k]);
    else
      w[k] = pack_bf16(v[2 * k], v[2 * k + 1]);
  }
  if (left >= 16 && vst == 32) {
#pragma unroll
    for (int k = 0; k < W; k += 8)
      asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(reinterpret_cast<uint32_t*>(dst) + k),
                   "r"(w[k]), "r"(w[k + 1]), "r"(w[k + 2]), "r"(w[k + 3]), "r"(w[k + 4]), "r"(w[k + 5]), "r"(w[k + 6]),
                   "r"(w[k + 7])
                   : "memory");
  } else if (left >= 16 && vst == 16) {
#pragma unroll
    for (int k = 0; k < W; k += 4)
      *reinterpret_cast<uint4*>(reinterpret_cast<uint32_t*>(dst) + k) = make_uint4(w[k], w[k + 1], w[k + 2], w[k + 3]);
  } else {
#pragma unroll
    for (int k = 0; k < 16; ++k)
      if (k < left) dst[k] = from_f32<T>(v[k]);
  }
}

// the product list of PA x PB pieces, smallest terms first
template <int PA, int PB>
struct Products;
template <>
struct Products<3, 3> {
  static constexpr int n = 6;
  __device__ static constexpr int a(int i) { return i == 0 ? 2 : (i == 1 ? 0 : (i == 2 ? 1 : (i == 3 ? 1 : 0))); }
  __device__ static constexpr int b(int i) { return i == 0 ? 0 : (i == 1 ? 2 : (i == 2 ? 1 : (i == 3 ? 0 : (i == 4 ? 1 : 0)))); }
};
template <>
struct Products<1, 3> {
  static constexpr int n = 3;
  __device__ static constexpr int a(int) { return 0; }
  __device__ static constexpr int b(int i) { return 2 - i; }
};
template <>
struct Products<1, 1> {
  static constexpr int n = 1;
  __device__ static constexpr int a(int) { return 0; }
  __device__ static constexpr int b(int) { return 0; }
};

// The groups in shared memory: units of group g are [pre[g], pre[g + 1]), its rows [lo[g], hi[g]) of `order`.
struct Groups {
  int *pre, *lo, *hi;
  int* bounds;  // this CTA's units
  static constexpr int INTS = 3 * MACE_SPECIES_MAX_GROUPS + 4;
  __device__ __forceinline__ explicit Groups(void* at)
      : pre(static_cast<int*>(at)),
        lo(pre + MACE_SPECIES_MAX_GROUPS + 2),
        hi(lo + MACE_SPECIES_MAX_GROUPS),
        bounds(hi + MACE_SPECIES_MAX_GROUPS) {}
};

// ------------------------------------------------------------------ layout
template <typename T, bool VEC>
struct Sl {
  static constexpr int P = sizeof(T) == 4 ? 3 : 1;  // pieces of a value
  static constexpr bool LONG = P == 1;              // sums of a whole tile (the result is rounded to 8 bits)
  static constexpr int PITCH = 128 + (VEC ? 0 : 16);  // of a ring unit: 32 rows x 128 bytes
  static constexpr int UPC = SL_KC * (int)sizeof(T) / 128;  // ring units per step of 64
  static constexpr int NU = 5;
  static constexpr int UNIT = 32 * PITCH;
  static constexpr int MAX_SLOTS = 8;
  static constexpr int OFF_A = (P == 3 ? 6 : 4) * SL_IMG;  // after the weight images
  static constexpr int STG = 32 * 128;                     // an epilogue warp's staging, 32 rows x 128 bytes
  static constexpr int OFF_STG = OFF_A + 4 * NU * UNIT;
  static constexpr int OFF_MIS = OFF_STG + 8 * STG;  // per ring unit and row: misalignment
  static constexpr int OFF_PRE = OFF_MIS + (VEC ? 0 : 4 * NU * 32);
  static constexpr int OFF_BAR = OFF_PRE + Groups::INTS * 4;
  static constexpr int NBAR = 8 + 2 * MAX_SLOTS + 1;
  static constexpr int BYTES = OFF_BAR + NBAR * 8 + 32;
  static_assert(BYTES <= 232448, "shared memory of a CTA");
};

// x k / n; 64-bit division is slow
__device__ __forceinline__ int64_t part(int64_t x, int k, int n) {
  return x < (1 << 22) && n < (1 << 10) ? (int64_t)((uint32_t)x * (uint32_t)k / (uint32_t)n) : x * k / n;
}

// Fills them, by the whole CTA (G <= 512 threads), and finds this CTA's units [t0, t1): the share-th of `shares`
// of the whole, or of min(shares, units) with `each` (no share without a unit between two that have some).  `start`:
// what a group costs beside its units, in half units (once for each of `runs` equal runs of its units); shares are
// equal in that sum, floor(share * sum / shares) on.
template <int THREADS>
__device__ __forceinline__ void load_groups(const SlParams& p, int unit_rows, int runs, int start, int share,
                                            int shares, bool each, const Groups& q, int64_t* warp_sums) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int64_t s = 0, mine = 0, per = 0;  // units of the groups up to this one, its own, those of a run
  int some = 0;  // groups up to this one that have rows
  if (tid < p.G) {
    const Range r = group_range(p.offsets, tid, p.n);
    q.lo[tid] = (int)r.lo;
    q.hi[tid] = (int)r.hi;
    per = ((r.hi - r.lo) * p.d + unit_rows - 1) / unit_rows;
    s = mine = per * runs;
  }
  const unsigned have = __ballot_sync(0xffffffffu, mine > 0);
  some = __popc(have & (0xffffffffu >> (31 - lane)));
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += u;
  }
  if (lane == 31) warp_sums[warp] = s;
  if (lane == 31) warp_sums[32 + warp] = some;
  if (tid < 2) q.bounds[tid] = 0;
  __syncthreads();
  int64_t all = 0, all_some = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) {
      s += warp_sums[w];
      some += (int)warp_sums[32 + w];
    }
    all += warp_sums[w];
    all_some += warp_sums[32 + w];
  }
  if (tid < p.G) q.pre[tid + 1] = (int)min(s, (int64_t)INT32_MAX);  // beyond it: offsets that overlap
  if (tid == 0) q.pre[0] = 0;
  const int scale = start ? 2 : 1;
  const int64_t cost = scale * all + (int64_t)start * runs * all_some;
  if (each) shares = (int)min((int64_t)shares, all);
  if (mine > 0 && share < shares) {
    // the group in which a bound lies says which unit it is
    const int64_t c0 = scale * (s - mine) + (int64_t)start * runs * (some - 1);  // where the group starts
    const int64_t len = scale * per + start;                                      // of a run
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int64_t x = part(cost, share + k, shares) - c0;
      if (x >= 0 && x < len * runs) {
        const int run = runs == 1 ? 0 : (int)(x / len);
        const int64_t unit = s - mine + run * per + (max(x - run * len - start, (int64_t)0) + scale - 1) / scale;
        q.bounds[k] = (int)min(unit, (int64_t)INT32_MAX);
      }
    }
    if (share + 1 == shares && s == all) q.bounds[1] = (int)min(all, (int64_t)INT32_MAX);
  }
  __syncthreads();
}

// Weight gradient: the shares of every group, for the join.  Share of unit u: the largest s with
// floor(s all / shares) <= u.
template <int THREADS>
__device__ __forceinline__ void write_spans(const SlParams& p, const Groups& q) {
  const int64_t all = q.pre[p.G];
  const int shares = (int)min((int64_t)p.shares, all);
  auto share_of = [&](int64_t u) -> int {
    const int64_t x = (u + 1) * shares - 1;
    return min(x <= UINT32_MAX ? (int)((uint32_t)x / (uint32_t)all) : (int)(x / all), shares - 1);
  };
  for (int g = threadIdx.x; g < p.G; g += THREADS) {
    const int64_t u0 = q.pre[g], u1 = q.pre[g + 1];
    int span = -1;
    if (u0 < u1) {
      const int s0 = share_of(u0);
      span = s0 | (s0 * all < u0 * shares) << 15 | share_of(u1 - 1) << 16;  // (u0 > floor(s0 all / shares))
    }
    p.spans[g] = span;
  }
}

// The steps of a CTA, in order; every role walks the same ones, holding little (the rest is in shared memory).
// Map: tiles t of (group, column tile, row tile).  Weight gradient: 64-row units t of the groups.
struct Walk {
  int t, g;
  __device__ __forceinline__ void init(const SlParams& p, const Groups& q, int t0) {
    t = t0;
    int lo = 0, hi = p.G - 1;  // the largest g with pre[g] <= t: empty groups have pre[g] == pre[g + 1]
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (q.pre[mid] <= t)
        lo = mid;
      else
        hi = mid - 1;
    }
    g = lo;
  }
  __device__ __forceinline__ void next(const Groups& q, int t1) {
    if (++t < t1)
      while (q.pre[g + 1] <= t) ++g;
  }
};

// Map: a tile's rows [at, end) of the grouped list (components counted), its column tile, and how many tiles of the
// same (group, column tile) are left with it.
struct Tile {
  int at, end;
  int ct, run;
  __device__ __forceinline__ Tile(const SlParams& p, const Groups& q, const Walk& w) {
    at = q.lo[w.g] * p.d;
    end = q.hi[w.g] * p.d;
    const int n_rt = (end - at + 127) >> 7;
    int rt = w.t - q.pre[w.g];
    ct = 0;
    if (p.n_ct > 1) {
      ct = rt / n_rt;
      rt -= ct * n_rt;
    }
    at += rt * 128;
    run = n_rt - rt;
  }
};

// A lane's row of the grouped list, loaded ahead of use.  The load is issued for every lane (from a clamped place)
// and its result first read by valid(): selecting a default right after the load would wait for it.
struct RowRef {
  int node, m;  // m < 0: no such row
  __device__ __forceinline__ void load(const SlParams& p, int at, int end) {
    const bool in = at < end;
    at = min(at, end - 1);
    int i = at;
    m = 0;
    if (p.d > 1) {
      i = __umulhi((uint32_t)at, p.div_mul) >> p.div_shift;
      m = at - i * p.d;
    }
    if (!in) m = -1;
    node = load_in(p.order + i);
  }
  __device__ __forceinline__ bool valid(const SlParams& p) const { return m >= 0 && node >= 0 && node < p.n; }
  __device__ __forceinline__ int64_t offset(const RowView& v) const { return node * v.sn + m * v.sm; }
  __device__ __forceinline__ uint32_t pieces(const RowView& v) const { return node * v.sn16 + m * v.sm16; }
};

constexpr uint32_t NO_ROW = 0xffffffffu;

// 32 row segments of 128 bytes.  Aligned rows: lane l copies 16-byte piece l % 8 of rows l / 8 + 4 i, whose offsets
// (in 16 bytes) it holds in off[i], piece j of row r to j ^ (r & 7).
__device__ __forceinline__ void spread_rows(uint32_t mine, uint32_t* off) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < 8; ++i) off[i] = __shfl_sync(0xffffffffu, mine, i * 4 + (lane >> 3));
}

// `at`: first byte of the segment within its row.  Rows are whole 16-byte pieces here: a copy whose source size is a
// register costs several instructions more than one that is all or nothing.
__device__ __forceinline__ void fetch_vec(uint32_t dst, const char* data, const uint32_t* off, int at, int row_bytes) {
  const int lane = threadIdx.x & 31, j = lane & 7, r0 = lane >> 3;
  const bool past = at + 16 * j >= row_bytes;
  const char* const src = past ? data : data + at + 16 * j;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = i * 4 + r0;
    cp_async16_or_zero(dst + r * 128 + ((j ^ (r & 7)) << 4), src + (uint64_t)off[i] * 16, past);
  }
}

// Rows of any alignment: the 16-byte pieces that contain the segment; mis[r]: where it starts in the first.  (Value by
// value, as the weight gradient takes rows of 4-byte values, costs the four warps here more than the shifting: 600 000
// fp32 rows 97 -> 61 164 us against 139.)  row: this lane's row.
template <int PITCH>
__device__ __forceinline__ void fetch_any(uint32_t dst, const char* data, const char* row, int at, int row_bytes,
                                          uint8_t* mis) {
  const int lane = threadIdx.x & 31;
  // copies of no bytes still name an aligned address
  const char* const dummy = reinterpret_cast<const char*>(reinterpret_cast<uint64_t>(data) & ~(uint64_t)15);
  const int seg = max(min(row_bytes - at, 128), 0);  // bytes of a row in this segment
  const uint64_t from = reinterpret_cast<uint64_t>(row + at);
  mis[lane] = (uint8_t)(from & 15);
#pragma unroll
  for (int i = 0; i < 9; ++i) {
    const int q = i * 32 + lane;
    const int r = q / 9, j = q - r * 9;
    const uint64_t f = __shfl_sync(0xffffffffu, from, r);
    const int left = (int)(f & 15) + seg - 16 * j;
    const uint32_t bytes = seg == 0 || left <= 0 ? 0u : (left < 16 ? (uint32_t)left : 16u);
    cp_async16(dst + r * PITCH + j * 16, bytes ? reinterpret_cast<const char*>((f & ~(uint64_t)15) + 16 * j) : dummy,
               bytes);
  }
}

// Map: 32 staged row segments of 128 bytes (piece j of row r at j ^ (r & 7)) to columns c0 .. c0 + left - 1 of their
// rows, one row per lane (mine: it exists).  Rows of any alignment: a row at a time, neighbouring lanes on
// neighbouring columns (not inlined: its registers would crowd the aligned path's).
template <typename T>
__device__ __noinline__ void copy_out_any(const SlParams& p, uint32_t stage_addr, int node, int m, bool mine, int c0,
                                          int left) {
  // (a shared-memory address: the compiler cannot see through the call that a pointer would be one)
  const uint8_t* const stage = static_cast<const uint8_t*>(__cvta_shared_to_generic(stage_addr));
  const int lane = threadIdx.x & 31;
  constexpr int CB = 128 / sizeof(T);  // columns of a segment
  if (p.out32) {
    const uint32_t o = mine ? node * p.out_n32 + m * p.out_m32 : NO_ROW;
    T* const to = static_cast<T*>(p.out) + c0 + lane;
    // (unrolled whole: the values of many rows are read before the first is stored.  600 000 bf16 rows of 97 -> 61,
    // fwd: 102 us, by 8 rows 134; fp32 dx: 138, by 8 146)
#pragma unroll
    for (int r = 0; r < 32; ++r) {
      const uint32_t ro = __shfl_sync(0xffffffffu, o, r);
#pragma unroll
      for (int c = 0; c < CB; c += 32) {
        const int byte = (c + lane) * (int)sizeof(T);
        const T v = load_as<T>(stage + r * 128 + ((((byte >> 4) ^ (r & 7)) << 4) | (byte & 15)));
        if (ro != NO_ROW && c + lane < left) to[ro + (uint32_t)c] = v;
      }
    }
  } else {
#pragma unroll 1
    for (int r = 0; r < 32; ++r) {
      const bool in = __shfl_sync(0xffffffffu, mine, r);
      const int64_t ro = __shfl_sync(0xffffffffu, node, r) * p.out_sn + __shfl_sync(0xffffffffu, m, r) * p.out_sm;
      for (int c = lane; c < left && c < CB; c += 32) {
        const int byte = c * (int)sizeof(T);
        if (in)
          (static_cast<T*>(p.out) + ro + c0)[c] =
              load_as<T>(stage + r * 128 + ((((byte >> 4) ^ (r & 7)) << 4) | (byte & 15)));
      }
    }
  }
}

template <typename T>
__device__ __forceinline__ void copy_out(const SlParams& p, const uint8_t* stage, const RowRef& ref, bool mine, int c0,
                                         int left) {
  int row = threadIdx.x & 31;
  asm volatile("" : "+r"(row));  // addresses are made here each time: held across the tiles they crowd the registers
  __syncwarp();
  if (p.vst) {
    // 4 rows x 128 bytes per instruction
    const uint32_t o = mine ? ref.node * p.out_n32 + ref.m * p.out_m32 : NO_ROW;
    const int j = row & 7;
    const bool have = left * (int)sizeof(T) > 16 * j;
    char* const to = static_cast<char*>(p.out) + (int64_t)c0 * sizeof(T) + 16 * j;
    const uint8_t* const src = stage + (row >> 3) * 128;
#pragma unroll
    for (int i0 = 0; i0 < 8; i0 += 4) {
      uint4 v[4];
      uint32_t ro[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // (r & 7 alternates between lane / 8 and lane / 8 + 4)
        v[i] = load_as<uint4>(src + (i0 + i) * 512 + ((j ^ ((row >> 3) + (i & 1) * 4)) << 4));
        ro[i] = __shfl_sync(0xffffffffu, o, (i0 + i) * 4 + (row >> 3));
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (ro[i] != NO_ROW && have) *reinterpret_cast<uint4*>(to + (uint64_t)ro[i] * 16) = v[i];
    }
  } else {
    copy_out_any<T>(p, tc::smem_u32(stage), ref.node, ref.m, mine, c0, left);
  }
  __syncwarp();
}

// Infinities and NaN among split operands: a piece of an infinity is inf - inf, so whatever it enters is NaN, and an
// infinite piece times a zero one is too: a whole row of results, or a column of them.  So a CTA that has met such a row,
// or weights that are not finite, goes over its results once more when it is done, and makes those that are NaN from
// the operands as they are, in fp32.  (A look at every result, or the call within the epilogue, cost 2 to 3 us of 125.
// 600 000 rows 128 -> 128 with one infinity among them take 0.7 ms, all of them NaN 1.5, all infinite 13, with a NaN or
// an infinity among the weights up to 11 and 39; the weight gradient up to 16, 0.4 and 24.)

// Map: this CTA's tiles, each by the epilogue warps that stored it
template <typename S>
__device__ __noinline__ void redo_map(const SlParams& p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  const Groups q(smem + S::OFF_PRE);
  const int t0 = q.bounds[0], t1 = q.bounds[1];
  const int lane = threadIdx.x & 31, quad = (threadIdx.x >> 5) & 3, half = (threadIdx.x >> 7) & 1, CW = p.NT / 2;
  const int64_t wk = p.transposed ? 1 : p.N, wc = p.transposed ? p.K : 1;
  Walk w;
  w.init(p, q, t0);
#pragma unroll 1
  for (; w.t < t1; w.next(q, t1)) {
    const Tile t(p, q, w);
    const int c0 = t.ct * p.NT + half * CW, c1 = min(c0 + CW, p.N);
    const float* const wt = static_cast<const float*>(p.w) + (int64_t)w.g * p.K * p.N;
    RowRef ref;  // lane r: row 32 quad + r
    ref.load(p, t.at + quad * 32 + lane, t.end);
    const bool mine = ref.valid(p);
    const int64_t at = mine ? ref.node * p.out_sn + ref.m * p.out_sm : -1;
    unsigned left = 0;  // rows with a NaN in these columns
#pragma unroll 8
    for (int r = 0; r < 32; ++r) {
      const int64_t to = __shfl_sync(0xffffffffu, at, r);
      const float* const y = static_cast<const float*>(p.out) + to;
      bool nan = false;
#pragma unroll
      for (int c = c0 + lane; c < c0 + 64; c += 32)
        if (to >= 0 && c < c1) nan |= y[c] != y[c];
      left |= (unsigned)__any_sync(0xffffffffu, nan) << r;
    }
    for (; left; left &= left - 1) {
      const int r = __ffs(left) - 1;
      const int64_t from = __shfl_sync(0xffffffffu, mine ? ref.offset(p.a) : 0, r);
      const float* const x = reinterpret_cast<const float*>(p.a.data + from);
      float* const y = static_cast<float*>(p.out) + __shfl_sync(0xffffffffu, at, r);
      bool nan = false;  // a NaN in the row: every result is one
      for (int k = lane; k < p.K; k += 32) nan |= x[k] != x[k];
      if (__any_sync(0xffffffffu, nan)) continue;
      for (int c = c0 + lane; c < c1; c += 32) {
        if (y[c] == y[c]) continue;
        float sum = 0.f;
        for (int k = 0; k < p.K && sum == sum;)
#pragma unroll 8
          for (const int e = min(k + 32, p.K); k < e; ++k) sum = __fmaf_rn(x[k], wt[k * wk + c * wc], sum);
        y[c] = p.alpha * sum;
      }
    }
  }
}

// Weight gradient: a lane's NT / 2 sums of row kl of a 128 x NT tile (columns c0 ..), done with group g: dW itself
// where this share held the whole group, else a partial tile: a share has two for each tile of the matrix, one for a
// group that begins with it or before it, one for a group that begins inside it (`inside`) and goes on.  A partial tile
// is stored as [column quad][row], so that a warp's 32 rows are one line per instruction.
template <typename T>
__device__ __forceinline__ void finish_wgrad(const SlParams& p, float* acc, int g, bool whole, bool inside, int tile,
                                             int share, int k0, int n0, int kl, int c0, int CW) {
  if (!whole) {
    float4* dst = reinterpret_cast<float4*>(p.part) + (((int64_t)tile * p.shares + share) * 2 + inside) * 32 * p.NT +
                  c0 / 4 * 128 + kl;
#pragma unroll
    for (int b = 0; b < 16; ++b)
      if (b * 4 < CW) dst[b * 128] = make_float4(acc[4 * b], acc[4 * b + 1], acc[4 * b + 2], acc[4 * b + 3]);
  } else if (k0 + kl < p.K) {
    T* dst = static_cast<T*>(p.out) + ((int64_t)g * p.K + k0 + kl) * p.N + n0 + c0;
    const int left = p.N - n0 - c0;
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      if (b * 16 >= CW) break;
#pragma unroll
      for (int k = 0; k < 16; ++k) acc[b * 16 + k] *= p.alpha;
      if (left - b * 16 > 0) store16<T>(dst + b * 16, acc + b * 16, left - b * 16, p.vst);
    }
  }
}

// Map: zeros in the rows outside every group, shared by warps 5 to 7 of every CTA.
template <typename T>
__device__ __forceinline__ void zero_rows(const SlParams& p) {
  const int lane = threadIdx.x & 31, w = (threadIdx.x >> 5) - 5;
  const int64_t b0 = min(max((int64_t)p.offsets[0], (int64_t)0), p.n);
  const int64_t b1 = max(min(max((int64_t)p.offsets[p.G], (int64_t)0), p.n), b0);
  const int64_t outside = (p.n - (b1 - b0)) * p.d;
  T* out = static_cast<T*>(p.out);
  for (int64_t r = blockIdx.x * (int64_t)3 + w; r < outside; r += (int64_t)gridDim.x * 3) {
    int64_t i = r / p.d;
    const int m = (int)(r - i * p.d);
    if (i >= b0) i += b1 - b0;
    const int64_t node = p.order[i];
    if (node < 0 || node >= p.n) continue;
    for (int c = lane; c < p.N; c += 32) out[node * p.out_sn + m * p.out_sm + c] = from_f32<T>(0.f);
  }
}

// 16 bytes at byte offset s of the 32 bytes (a, b)
__device__ __forceinline__ uint4 shifted(uint4 a, uint4 b, int s) {
  uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  if (s & 8) {
#pragma unroll
    for (int k = 0; k < 6; ++k) w[k] = w[k + 2];
  }
  if (s & 4) {
#pragma unroll
    for (int k = 0; k < 5; ++k) w[k] = w[k + 1];
  }
  const int bits = 8 * (s & 3);
  return make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits),
                    __funnelshift_r(w[2], w[3], bits), __funnelshift_r(w[3], w[4], bits));
}

// 8 K-values of row n of a B image: their bf16 pieces, `piece` bytes apart
template <int P>
__device__ __forceinline__ void put_eight(uint8_t* img, int piece, int n, int chunk, const float* v) {
  uint32_t t[4][3];
#pragma unroll
  for (int q = 0; q < 4; ++q) split2<P>(v[2 * q], v[2 * q + 1], t[q]);
#pragma unroll
  for (int b = 0; b < P; ++b)
    store_piece(img + b * piece + n * 128 + ((chunk ^ (n & 7)) << 4), t[0][b], t[1][b], t[2][b], t[3][b]);
}

// Map: the weight images of steps [k0, k0 + nk) of (group g, column tile ct), at img0 + step * stride, by warps
// 4 to 7; full: the first step's barrier (arrived on as each step is done).  A round is 64 image rows of a step:
// 16 items of 32 (image row, K octet) pairs, one per lane, four items per warp, with all of their loads in flight
// (through shared memory by cp.async, rewritten in place, was slower: 40 000 fp32 rows 128 -> 128 20.6 us, 19.0 so).
// Weights (K, N): an item is one octet of 32 neighbouring columns; transposed (N, K): 8 octets of 4 rows.
template <typename T, int PB>
__device__ __forceinline__ void fill_weights(const SlParams& p, uint8_t* img0, int stride, int g, int ct, int k0,
                                             int nk, uint32_t full, volatile int* odd) {
  const int lane = threadIdx.x & 31, w4 = (threadIdx.x >> 5) & 3;
  const int NT = p.NT;
  const T* wt = static_cast<const T*>(p.w) + (int64_t)g * p.K * p.N;
  float probe = 0.f;
#pragma unroll 1
  for (int s = 0; s < nk; ++s) {
    uint8_t* const img = img0 + s * stride;
#pragma unroll 1
    for (int h = 0; h * 64 < NT; ++h) {
      float v[4][8];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int j = h * 16 + u * 4 + w4;
        const int n = p.transposed ? j * 4 + (lane >> 3) : (j >> 3) * 32 + lane, kk = (p.transposed ? lane & 7 : j & 7) * 8;
        const int col = ct * NT + n, k = (k0 + s) * SL_KC + kk;
        const bool in = n < NT && col < p.N;
        if (p.transposed && p.w_vec) {
          if (in && k + 8 <= p.K) {
            load_eight(reinterpret_cast<const uint8_t*>(wt + (int64_t)col * p.K + k), v[u], T{});
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[u][e] = in && k + e < p.K ? to_f32(wt[(int64_t)col * p.K + k + e]) : 0.f;
          }
        } else {
          const T* src = p.transposed ? wt + (int64_t)col * p.K + k : wt + (int64_t)k * p.N + col;
          const int64_t step = p.transposed ? 1 : p.N;
#pragma unroll
          for (int e = 0; e < 8; ++e) v[u][e] = in && k + e < p.K ? to_f32(src[e * step]) : 0.f;
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int j = h * 16 + u * 4 + w4;
        const int n = p.transposed ? j * 4 + (lane >> 3) : (j >> 3) * 32 + lane;
        if constexpr (PB == 3) {
#pragma unroll
          for (int e = 0; e < 8; ++e) probe = __fmaf_rn(v[u][e], 0.f, probe);
        }
        if (n < NT) put_eight<PB>(img, p.img, n, p.transposed ? lane & 7 : j & 7, v[u]);
      }
    }
    if (PB == 3 && probe != 0.f) *odd = 1;
    tc::fence_proxy_async();
    warp_arrive(full + 8 * s);
  }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(SL_THREADS, 1) k_species_map(const __grid_constant__ SlParams p) {
  using S = Sl<T, VEC>;
  constexpr int P = S::P, NU = S::NU;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = tc::smem_u32(smem);
  const Groups q(smem + S::OFF_PRE);
  uint64_t* const bars = reinterpret_cast<uint64_t*>(smem + S::OFF_BAR);
  uint32_t* const tslot = reinterpret_cast<uint32_t*>(bars + S::NBAR);
  volatile int* const abort = reinterpret_cast<int*>(tslot + 1);
  volatile int* const odd = reinterpret_cast<int*>(tslot + 2);  // a weight or a row is not finite
  auto bar = [&](int i) { return tc::smem_u32(bars + i); };
  auto A_FULL = [&](int s) { return bar(s); };
  auto A_FREE = [&](int s) { return bar(2 + s); };
  auto D_FULL = [&](int s) { return bar(4 + s); };
  auto D_FREE = [&](int s) { return bar(6 + s); };
  auto B_FULL = [&](int s) { return bar(8 + s); };
  auto B_FREE = [&](int s) { return bar(8 + S::MAX_SLOTS + s); };
  const uint32_t DONE = bar(8 + 2 * S::MAX_SLOTS);
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // known to be uniform

  if (base & 1023u) {  // the images need 1024-byte alignment
    if (tid == 0) atomicExch(&g_species_error, TC_ERR_ALIGN);
    return;
  }

  const int NT = p.NT;
  if (warp == 15) {  // while the others wait for the offsets
    if (lane == 0) {
      *abort = *odd = 0;
      for (int s = 0; s < 2; ++s) {
        tc::mbar_init(A_FULL(s), 4);
        tc::mbar_init(A_FREE(s), 1);
        tc::mbar_init(D_FULL(s), 1);
        tc::mbar_init(D_FREE(s), 8);
      }
      for (int s = 0; s < S::MAX_SLOTS; ++s) {
        tc::mbar_init(B_FULL(s), 4);
        tc::mbar_init(B_FREE(s), 1);
      }
      tc::mbar_init(DONE, 1);
      tc::fence_barrier_init();
    }
    __syncwarp();
    tc::tmem_alloc(tc::smem_u32(tslot), SL_TMEM);
    tc::tmem_relinquish();
  }
  pdl_wait();  // nothing of the caller's is read or written before
  tc::fence_before_sync();
  // unit: a row tile of a (group, column tile)
  load_groups<SL_THREADS>(p, 128, p.n_ct, p.start, blockIdx.x, gridDim.x, false, q, reinterpret_cast<int64_t*>(smem));
  tc::fence_after_sync();
  const int t0 = q.bounds[0], t1 = q.bounds[1];
  if (t0 >= t1) {
    if (warp >= 5 && warp < 8) zero_rows<T>(p);
    if (warp == 15) tc::tmem_dealloc(SL_D, SL_TMEM);
    return;
  }
  const int n_k = (p.K + SL_KC - 1) / SL_KC;  // steps of a tile
  const bool resident = n_k <= p.slots;       // the weight images of a tile stay for the next row tile
  const uint32_t tmem = SL_D;  // an allocation of all 512 columns starts at column 0

  if (warp < 4) {
    // ---------------- operand A: memory -> ring -> registers -> TMEM ----------------
    const uint32_t ring = base + S::OFF_A + warp * NU * S::UNIT;
    uint8_t* const mis = smem + S::OFF_MIS + warp * NU * 32;
    const int row_bytes = p.a.width * (int)sizeof(T);
    const uint32_t tq = tmem + ((uint32_t)(warp * 32) << 16) + SL_A;
    // the fetching side runs NU - 1 units ahead; the atoms of its rows are loaded one tile before
    const int tile_units = n_k * S::UPC;  // ring units of a tile
    const int units = (t1 - t0) * tile_units;
    int left = units, fu = 0, slot_f = 0;  // units to fetch, unit within the tile, ring slot
    RowRef ref;  // this lane's row of the next tile
    Walk w_tile;
    uint32_t off[8];
    const char* row = nullptr;
    auto load_tile = [&]() {
      const Tile t(p, q, w_tile);
      ref.load(p, t.at + warp * 32 + lane, t.end);
    };
    auto fetch = [&]() {
      if (left > 0) {
        --left;
        if (fu == 0) {
          // (a row outside the tile may hold anything, as its TMEM lane is never stored: it stands for row 0)
          const bool ok = ref.valid(p);
          if constexpr (VEC)
            spread_rows(ok ? ref.pieces(p.a) : 0u, off);
          else
            row = p.a.data + (ok ? ref.offset(p.a) : 0);
          w_tile.next(q, t1);
          if (w_tile.t < t1) load_tile();
        }
        const uint32_t dst = ring + slot_f * S::UNIT;
        if constexpr (VEC)
          fetch_vec(dst, p.a.data, off, fu * 128, row_bytes);
        else
          fetch_any<S::PITCH>(dst, p.a.data, row, fu * 128, row_bytes, mis + slot_f * 32);
        slot_f = slot_f + 1 == NU ? 0 : slot_f + 1;
        if (++fu == tile_units) fu = 0;
      }
      cp_commit();
    };
    w_tile.init(p, q, t0);
    load_tile();
    // (one loop, so that the code of a unit exists once: the roles' loops together fill the instruction cache)
    int slot = 0;
    bool ok = true;
#pragma unroll 1
    for (int i = 1 - NU; i < units && ok; ++i) {
      const int it = i / S::UPC, u = i - it * S::UPC, s = it & 1;
      if (i >= 0) cp_wait<NU - 2>();
      __syncwarp();
      fetch();
      if (i < 0) continue;
      const uint8_t* const src = smem + S::OFF_A + (warp * NU + slot) * S::UNIT;
      const uint8_t* const ms = mis + slot * 32;
      slot = slot + 1 == NU ? 0 : slot + 1;
      if (u == 0) {
        ok = it < 2 || wait_phase(A_FREE(s), ((it >> 1) - 1) & 1, abort);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc::fence_after_sync();
      }
      const uint32_t ta = tq + s * (P * 32);
      // this lane's row: 128 bytes of it
      const int sh = VEC ? 0 : ms[lane];
      auto piece = [&](int j) { return load_as<uint4>(src + lane * S::PITCH + (VEC ? j ^ (lane & 7) : j) * 16); };
      uint32_t out[P][16];
      uint4 cur = piece(0);
#pragma unroll
      for (int h = 0; h < 8 / (P == 3 ? 8 : 4); ++h) {
#pragma unroll
        for (int q = 0; q < (P == 3 ? 8 : 4); ++q) {
          const int j = h * 4 + q;
          uint4 v = cur;
          if constexpr (VEC) {
            if (j < 7) cur = piece(j + 1);
          } else {
            const uint4 nx = piece(j + 1);
            v = shifted(cur, nx, sh);
            cur = nx;
          }
          if constexpr (P == 3) {
            uint32_t t[3];
            split2<P>(__uint_as_float(v.x), __uint_as_float(v.y), t);
#pragma unroll
            for (int a = 0; a < P; ++a) out[a][2 * q] = t[a];
            split2<P>(__uint_as_float(v.z), __uint_as_float(v.w), t);
#pragma unroll
            for (int a = 0; a < P; ++a) out[a][2 * q + 1] = t[a];
          } else {
            out[0][4 * q] = v.x;
            out[0][4 * q + 1] = v.y;
            out[0][4 * q + 2] = v.z;
            out[0][4 * q + 3] = v.w;
          }
        }
        if constexpr (P == 1) tmem_st16u(ta + h * 16, out[0]);
      }
      if constexpr (P == 3) {
#pragma unroll
        for (int a = 0; a < P; ++a) tmem_st16u(ta + a * 32 + u * 16, out[a]);
      }
      if (u == S::UPC - 1) {
        tc::tmem_wait_st();
        tc::fence_before_sync();
        warp_arrive(A_FULL(s));
      }
    }
    cp_wait<0>();
  } else if (warp < 8) {
    // ---------------- operand B: the weight images, and the MMAs ----------------
    // MMAs of step `it` with the images of slot bs, by one elected thread; `use`: how often the slot was filled
    // before, or -1 when its images were there already.  The queue of issued MMAs is a few hundred cycles deep, so
    // the path from one step's last to the next step's first is kept short: two waits, no warp-wide operation.
    const uint32_t idesc = idesc_bf16(NT), bhi = (uint32_t)(tc::sw128_desc(base) >> 32);
    // The accumulator takes the sn-th sum: one step, or for bf16 (S::LONG) a whole tile, of which this is the first /
    // last.
    auto issue = [&](int it, int bs, int use, bool release, int sn, bool first, bool last) -> bool {
      using PR = Products<P, P>;
      const int s = it & 1;
      if (use >= 0 && !wait_phase(B_FULL(bs), use & 1, abort)) return false;
      if (!wait_phase(A_FULL(s), (it >> 1) & 1, abort)) return false;
      if (first && sn >= 2 && !wait_phase(D_FREE(sn & 1), ((sn >> 1) - 1) & 1, abort)) return false;
      tc::fence_after_sync();
      const uint32_t dcol = SL_D + (sn & 1) * 128;
      const uint32_t blo = (uint32_t)tc::sw128_desc(base + bs * (P * p.img));
      // (the stage as a constant: little is left to compute)
      auto emit = [&](auto stage) {
        constexpr uint32_t st = decltype(stage)::value;
#pragma unroll
        for (int q = 0; q < PR::n; ++q)
#pragma unroll
          for (int ks = 0; ks < SL_KC / 16; ++ks)
            mma_bf16_ta(dcol, SL_A + st * (P * 32) + PR::a(q) * 32 + ks * 8, blo + PR::b(q) * (p.img / 16) + ks * 2, bhi,
                        idesc, !first || q > 0 || ks > 0);
      };
      if (s)
        emit(std::integral_constant<uint32_t, 1>{});
      else
        emit(std::integral_constant<uint32_t, 0>{});
      tc::mma_commit(A_FREE(s));
      if (last) tc::mma_commit(D_FULL(sn & 1));
      if (release) tc::mma_commit(B_FREE(bs));
      return true;
    };
    bool ok = true;
    auto fill = [&](int g, int ct, int k0, int nk, int slot0) {
      fill_weights<T, P>(p, smem + slot0 * P * p.img, P * p.img, g, ct, k0, nk, bar(8 + slot0), odd);
    };
    Walk w;
    w.init(p, q, t0);
    int it = 0, tile_no = 0, fills = 0;  // steps, tiles; image sets (resident) or images written
    while (w.t < t1 && ok) {
      const Tile t(p, q, w);
      if (resident) {
        // the tiles of this CTA that share the weights
        const int run = min(t.run, t1 - w.t);
        for (int k = 0; k < n_k && ok && fills > 0; ++k) ok = wait_phase(B_FREE(k), (fills - 1) & 1, abort);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        fill(w.g, t.ct, 0, n_k, 0);
        if (warp == 4 && elect_one())
          for (int i = 0; i < run && ok; ++i)
            for (int k = 0; k < n_k && ok; ++k)
              ok = issue(it + i * n_k + k, k, i == 0 ? fills : -1, i + 1 == run,
                         S::LONG ? tile_no + i : it + i * n_k + k, !S::LONG || k == 0, !S::LONG || k + 1 == n_k);
        it += run * n_k;
        tile_no += run;
        ++fills;
        w.t += run - 1;
      } else {
        for (int k = 0; k < n_k && ok; ++k, ++it, ++fills) {
          const int s = fills % p.slots, use = fills / p.slots;
          ok = use == 0 || wait_phase(B_FREE(s), (use - 1) & 1, abort);
          ok = __all_sync(0xffffffffu, ok);
          if (ok) fill(w.g, t.ct, k, 1, s);
          if (ok && warp == 4 && elect_one())
            ok = issue(it, s, use, true, S::LONG ? tile_no : it, !S::LONG || k == 0, !S::LONG || k + 1 == n_k);
          ok = __all_sync(0xffffffffu, ok);
        }
        ++tile_no;
      }
      ok = __all_sync(0xffffffffu, ok);
      w.next(q, t1);
    }
    if (warp == 4) {
      if (elect_one()) {  // every MMA issued is complete (bounded)
        tc::mma_commit(DONE);
        tc::mbar_wait(DONE, 0);
      }
      __syncwarp();
    } else {
      zero_rows<T>(p);
    }
  } else {
    // ---------------- epilogue ----------------
    const int quad = warp & 3, half = (warp - 8) >> 2;
    const int CW = NT / 2;  // columns of this warp: 16, 32, 48 or 64
    const uint32_t tq = tmem + ((uint32_t)(quad * 32) << 16) + SL_D + half * CW;
    uint8_t* const stage = smem + S::OFF_STG + (warp - 8) * S::STG;
    Walk w;
    w.init(p, q, t0);
    float acc[64];
    bool ok = true;
    bool fresh = true;   // acc holds nothing yet
    float probe = 0.f;   // NaN once a row was not finite (its first result tells)
    RowRef ref{-1, -1};  // this lane's row of the tile, loaded while the tile is computed
    int ct = 0, k = 0;   // the tile's column tile, the step
    for (int sn = 0; w.t < t1 && ok; ++sn) {
      const int s = sn & 1;
      if (fresh) {
        const Tile t(p, q, w);
        ref.load(p, t.at + quad * 32 + lane, t.end);
        ct = t.ct;
      }
      ok = wait_phase(D_FULL(s), (sn >> 1) & 1, abort);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc::fence_after_sync();
      const uint32_t td = tq + s * 128;
      if (fresh) {
#pragma unroll
        for (int k = 0; k < 64; ++k) acc[k] = 0.f;
      }
      // (alpha meets the sums of a step: with the weights, before they are split, it left the range of fp32 where the
      // result does not)
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        uint32_t v[16];
        if (h * 16 < CW) tmem_ld16u(td + h * 16, v);
        tc::tmem_wait_ld();
        if (h == 3) {
          tc::fence_before_sync();
          warp_arrive(D_FREE(s));
        }
#pragma unroll
        for (int k = 0; k < 16; k += 2) fma2(acc[h * 16 + k], acc[h * 16 + k + 1], v[k], v[k + 1], p.alpha);
      }
      fresh = false;
      k += S::LONG ? n_k : 1;
      if (k < n_k) continue;
      k = 0;
      const int c0 = ct * NT + half * CW;
      // Rows leave through shared memory, CB columns at a time: a thread holds one row, and 32-byte stores of it
      // touch 32 rows per instruction (600 000 rows 128 -> 128 fp32: 149 us with them, 130 staged).
      constexpr int CB = 128 / sizeof(T);  // columns of a 128-byte row segment
      const bool mine = ref.valid(p);
      if (P == 3 && mine) probe = __fmaf_rn(acc[0], 0.f, probe);
#pragma unroll
      for (int b = 0; b < 64; b += CB) {
        const int left = min(p.N - c0 - b, CW - b);  // columns of this segment
        if (left <= 0) break;
        // piece j of row r at j ^ (r & 7); the addresses are made here each time: held across the tiles they
        // would push the accumulators to memory
        int row = lane;
        asm volatile("" : "+r"(row));
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          uint32_t w4[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            if constexpr (sizeof(T) == 4)
              w4[q] = __float_as_uint(acc[b + 4 * j + q]);
            else
              w4[q] = pack_bf16(acc[b + 8 * j + 2 * q], acc[b + 8 * j + 2 * q + 1]);
          }
          store_piece(stage + row * 128 + ((j ^ (row & 7)) << 4), w4[0], w4[1], w4[2], w4[3]);
        }
        __syncwarp();
        copy_out<T>(p, stage, ref, mine, c0 + b, left);
        __syncwarp();
      }
      fresh = true;
      w.next(q, t1);
    }
    if (P == 3 && probe != 0.f) *odd = 1;
  }
  tc::fence_before_sync();
  __syncthreads();
  if (tid == 0 && *abort) atomicExch(&g_species_error, TC_ERR_TIMEOUT);
  if constexpr (P == 3)
    if (*odd && !*abort && threadIdx.x >= 256) redo_map<S>(p);
  if (warp == 15) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, SL_TMEM);
  }
}

// launches a kernel with `smem` bytes of dynamic shared memory; attr_set: of this kernel, per device (the attribute
// call is slow on the host)
template <typename K>
int launch_big(const char* name, K kernel, bool* attr_set, int grid, int threads, int smem, cudaStream_t s,
               const SlParams& p) {
  int dev = 0;
  MACE_CUDA_TRY(cudaGetDevice(&dev));
  if (dev >= 64 || !attr_set[dev]) {
    MACE_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    if (dev < 64) attr_set[dev] = true;
  }
  return launch(name, kernel, grid, threads, smem, s, p);
}

}  // namespace

}  // namespace mace

#include "species_direct.cuh"
#include "species_wgrad.cuh"

namespace mace {

namespace {

// dW of the groups that several shares hold, in share order, and of empty groups (zero).  CTA (g, y, tile): group g,
// rows 8 (y % 16) .. of the tile, in blocks of 8 rows x 8 column quads (64 lanes).  Few shares: the four sets of 64
// threads of the CTAs with y < 16 take a block each; many: CTA y takes block y / 16 (of more than 16 groups, which mostly
// have few shares, all blocks), each set every fourth share.  Eight loads in flight per thread need its 64 registers
// (weight gradients of 40 000 rows 128 x 128 in 4 groups: 20.8 us, 21.8 with 40 registers, 32.6 with one set per block;
// of 60 000 rows in 89 groups 28.4, 29.8 with a CTA per block).
template <typename T>
__global__ void __launch_bounds__(256, 4) k_species_wgrad_join(const __grid_constant__ SlParams p) {
  pdl_wait();
  __shared__ float4 part[4][64];
  const int g = blockIdx.x, tid = threadIdx.x;
  const int span = p.spans[g];
  const int s0 = span & 0x7fff, s1 = span >> 16;  // shares of the group; none: s1 = -1
  if (s0 == s1) return;                           // written by its only share
  const int lane = tid & 63, sl = tid >> 6;
  const int kl = (blockIdx.y & 15) * 8 + (lane & 7), block = blockIdx.y >> 4, blocks = gridDim.y >> 4;
  const int tiles = p.n_ct * p.n_kt;
  for (int tile = blockIdx.z; tile < tiles; tile += gridDim.z) {
    const int k0 = (tile / p.n_ct) * 128, n0 = (tile % p.n_ct) * p.NT;
    const float4* const first = reinterpret_cast<const float4*>(p.part) + (int64_t)tile * p.shares * 64 * p.NT + kl;
    const int inside = span & 0x8000 ? 32 * p.NT : 0;  // where its partial tile of share s0 is the second
    T* const row = static_cast<T*>(p.out) + ((int64_t)g * p.K + k0 + kl) * p.N + n0;
    auto sum = [&](int cq, int from, int step) {
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      const float4* at = first + (int64_t)from * 64 * p.NT + cq * 128;
      int skip = from == s0 ? inside : 0;
#pragma unroll 8
      for (int s = from; s <= s1; s += step, at += step * 64 * p.NT, skip = 0) {
        const float4 v = at[skip];
        acc.x += v.x;
        acc.y += v.y;
        acc.z += v.z;
        acc.w += v.w;
      }
      return acc;
    };
    auto write = [&](int cq, float4 a) {
      if (k0 + kl >= p.K) return;
      const float v[4] = {p.alpha * a.x, p.alpha * a.y, p.alpha * a.z, p.alpha * a.w};
      if (p.vst && n0 + cq * 4 + 4 <= p.N) {
        store4(row + cq * 4, v);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (n0 + cq * 4 + k < p.N) row[cq * 4 + k] = from_f32<T>(v[k]);
      }
    };
    if (s1 - s0 < 8) {
      const int cq = sl * 8 + (lane >> 3);
      if (block == 0 && cq * 4 < p.NT) write(cq, sum(cq, s0, 1));
      continue;
    }
    for (int b = block; b * 32 < p.NT; b += blocks) {
      const int cq = b * 8 + (lane >> 3);
      part[sl][lane] = sum(cq, s0 + sl, 4);
      __syncthreads();
      if (sl == 0) {
        float4 a = part[0][lane];
#pragma unroll
        for (int q = 1; q < 4; ++q) {
          a.x += part[q][lane].x;
          a.y += part[q][lane].y;
          a.z += part[q][lane].z;
          a.w += part[q][lane].w;
        }
        write(cq, a);
      }
      __syncthreads();
    }
  }
}

// ------------------------------------------------------------------ host side
bool bad_sizes(int32_t dtype, int64_t n, int32_t d, int32_t G, int32_t K, int32_t M) {
  return (dtype != MACE_F32 && dtype != MACE_BF16) || n < 0 || n > INT32_MAX || d < 1 || d > 1024 || G < 1 ||
         G > MACE_SPECIES_MAX_GROUPS || K < 1 || K > MACE_SPECIES_MAX_CHANNELS || M < 1 ||
         M > MACE_SPECIES_MAX_CHANNELS ||
         n * d > MACE_SPECIES_MAX_ROWS || (n * d + 63) / 64 + G > INT32_MAX / ((M + 31) / 32);
}

int sm_count() {
  static int count[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 148;
  if (dev >= 64) return 148;
  if (count[dev] == 0) {
    int v = 0;
    if (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || v < 1) v = 148;
    count[dev] = v;
  }
  return count[dev];
}

// columns of a tile: an even split of `cols` into multiples of 32, at most `most`
int tile_cols(int cols, int most) {
  const int tiles = (cols + most - 1) / most;
  return std::min(most, ((cols + tiles - 1) / tiles + 31) / 32 * 32);
}

int vector_bytes(const void* ptr, int64_t s0, int64_t s1, int64_t s2) {
  for (int v : {32, 16})
    if (reinterpret_cast<uintptr_t>(ptr) % v == 0 && s0 % v == 0 && s1 % v == 0 && s2 % v == 0) return v;
  return 0;
}

RowView row_view(const void* data, int64_t sn, int64_t sm, int width, int size) {
  return {static_cast<const char*>(data), sn * size, sm * size, width, (uint32_t)(sn * size / 16),
          (uint32_t)(sm * size / 16)};
}

// x / d for x < 2^31: x times ceil(2^(31 + s) / d), 2^(s - 1) < d <= 2^s, shifted by 31 + s
void set_divisor(SlParams* p, int d) {
  int s = 1;
  while ((1 << s) < d) ++s;
  p->div_mul = (uint32_t)((((uint64_t)1 << (31 + s)) + d - 1) / d);
  p->div_shift = s - 1;
}

// weight images of a step that fit the map's shared memory at NT columns and `pieces` pieces, and a piece's bytes
int image_slots(int NT, int pieces, int* img) {
  *img = NT > 64 ? SL_IMG : NT * 128;
  return std::min(8, (pieces == 3 ? 2 * 3 : 4) * SL_IMG / (pieces * *img));
}

bool aligned_rows(const RowView& v, int64_t n, int d, int size) {
  // (row offsets in 16 bytes fit 32 bits)
  return (reinterpret_cast<uintptr_t>(v.data) & 15) == 0 && v.width * size % 16 == 0 && (n <= 1 || v.sn % 16 == 0) && (d <= 1 || v.sm % 16 == 0) &&
         ((n - 1) * v.sn + (d - 1) * v.sm) / 16 < (int64_t)NO_ROW;
}

template <typename T, bool VEC>
int launch_map(const SlParams& p, int grid, cudaStream_t s) {
  static bool attr_set[64] = {};
  return launch_big("species_map", k_species_map<T, VEC>, attr_set, grid, SL_THREADS, Sl<T, VEC>::BYTES, s, p);
}

template <typename TA, typename T, bool VEC>
int launch_wgrad(const SlParams& p, int grid, cudaStream_t s) {
  static bool attr_set[64] = {};
  static int regs = 0;  // the shares that the kernel deals out are taken from what it is launched with
  if (regs == 0) {
    cudaFuncAttributes a;
    MACE_CUDA_TRY(cudaFuncGetAttributes(&a, k_species_wgrad<TA, T, VEC>));
    regs = a.numRegs;
  }
  if (regs != WG_REGS) return fail(MACE_ERR_CUDA, "species_wgrad: built with other than 80 registers a thread");
  return launch_big("species_wgrad", k_species_wgrad<TA, T, VEC>, attr_set, grid, WG_THREADS, Wg<TA, T, VEC>::BYTES, s, p);
}

// (one share has every group whole)
int64_t partial_bytes(const SlParams& p) {
  return p.shares > 1 ? (int64_t)p.n_ct * p.n_kt * p.shares * 2 * 128 * p.NT * 4 : 0;
}

// shares (CTAs along the rows) and tiles of a weight gradient
void wgrad_split(int64_t n, int32_t d, int32_t G, int32_t K, int32_t M, SlParams* p) {
  p->NT = tile_cols(M, 128);
  p->n_ct = (M + p->NT - 1) / p->NT;
  p->n_kt = (K + 127) / 128;
  const int64_t units = (n * d + SL_KC - 1) / SL_KC + std::min<int64_t>(G, n);
  const int tiles = p->n_ct * p->n_kt;
  p->shares = (int)std::max<int64_t>(1, std::min<int64_t>(units, (sm_count() + tiles - 1) / tiles));
  // The error of a sum grows with the square root of its steps, so long lists take more shares, each SM as many as the
  // others.  (MACE_SPECIES_MAX_ROWS rows make at most 16 533 shares; the join's table holds 32 767.)
  p->shares *= (int)std::max<int64_t>(1, (units + (int64_t)p->shares * SL_STEPS - 1) / ((int64_t)p->shares * SL_STEPS));
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
  if (unaligned(value_size(dtype), x, w, y) || unaligned(4, order, offsets))
    return fail(MACE_ERR_BAD_ARG, "mace_species_linear: an address is not a multiple of its values' size");
  if (n == 0) return MACE_OK;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int es = dtype == MACE_F32 ? 4 : 2;
  SlParams p{};
  p.a = row_view(x, xn, xm, K, es);
  p.w = w;
  p.transposed = transpose;
  p.out = y;
  p.out_sn = yn;
  p.out_sm = ym;
  // (as for the input: whole 16-byte pieces, offsets in 32 bits)
  const RowView out = row_view(y, yn, ym, M, es);
  p.vst = aligned_rows(out, n, d, es);
  p.out32 = (n - 1) * yn + (d - 1) * ym + M < (int64_t)NO_ROW;
  p.out_n32 = p.vst ? out.sn16 : (uint32_t)yn;
  p.out_m32 = p.vst ? out.sm16 : (uint32_t)ym;
  p.order = order;
  p.offsets = offsets;
  p.n = n;
  p.d = d;
  p.G = G;
  set_divisor(&p, d);
  p.K = K;
  p.N = M;
  p.w_vec = (transpose ? K : M) * es % 16 == 0 && reinterpret_cast<uintptr_t>(w) % 16 == 0;
  p.alpha = alpha;
  // direct: bf16 in whole pieces, nothing to convert (600 000 rows 128 -> 128: 57 us, 82 by the general kernel)
  const bool vec = aligned_rows(p.a, n, d, es), direct = dtype == MACE_BF16 && vec && p.w_vec;
  const int sms = sm_count();
  const int64_t row_tiles = (n * d + 127) / 128;
  // narrower column tiles while the row tiles leave SMs idle (3000 fp32 rows 128 -> 128: 9.3 us, 12.6 with tiles of
  // 128 columns; bf16 no difference)
  int most = 128;
  while (most > 32 && row_tiles * ((M + most - 1) / most) * 2 <= sms) most /= 2;
  // and so narrow that the weight images of the whole K stay in shared memory (K <= 512), rather than being made
  // anew for every tile (256 -> 256 fp32 channels, 300k rows: 326 us, 580 so)
  const int n_k = (K + SL_KC - 1) / SL_KC, pieces = dtype == MACE_F32 ? 3 : 1;
  if (!direct) {
    int fit = most;
    while (fit > 32 && n_k > image_slots(tile_cols(M, fit), pieces, &p.img)) fit /= 2;
    if (n_k <= image_slots(tile_cols(M, fit), pieces, &p.img)) most = fit;
  }
  p.NT = tile_cols(M, most);
  p.slots = image_slots(p.NT, pieces, &p.img);
  p.n_ct = (M + p.NT - 1) / p.NT;
  p.n_kt = 1;
  // Making a group's images costs about as much as 1.5 row tiles.  40 000 fp32 rows of 4 species 128 -> 128 21.2 us
  // without it, 18.5 with 4 or 6; 600 000 rows 128.5, 125.0 with 4, 124.6 with 6; 60 000 rows of 89 species 29.1, 26.5
  // with 4, 27.4 with 6.  bf16 rows copied as they lie (direct): no difference.
  p.start = !direct && n_k <= p.slots ? 4 : 0;
  const int grid = (int)std::min<int64_t>(sms, (row_tiles + std::min<int64_t>(G, n)) * p.n_ct);
  if (direct) return launch_direct<false>(p, grid, s);
  if (dtype == MACE_F32)
    return vec ? launch_map<float, true>(p, grid, s) : launch_map<float, false>(p, grid, s);
  return launch_map<bf16, false>(p, grid, s);
}

extern "C" int mace_species_linear_wgrad_workspace(int64_t n, int32_t d, int32_t G, int32_t K, int32_t M,
                                                   int64_t* bytes) {
  if (bad_sizes(MACE_F32, n, d, G, K, M) || !bytes)
    return fail(MACE_ERR_BAD_ARG, "mace_species_linear_wgrad_workspace: bad arguments");
  SlParams p{};
  wgrad_split(n, d, G, K, M, &p);
  *bytes = partial_bytes(p) + (int64_t)G * 4;
  return MACE_OK;
}

extern "C" int mace_species_linear_wgrad(int32_t dtype, const void* x, int64_t xn, int64_t xm, const float* xs,
                                         const void* dy, int64_t yn, int64_t ym, int32_t G, int32_t K, int32_t M,
                                         const int32_t* order, const int32_t* offsets, int64_t n, int32_t d,
                                         float alpha, void* dw, void* ws, int64_t ws_bytes, void* stream) {
  if (bad_sizes(dtype, n, d, G, K, M) || xn < 0 || xm < 0 || yn < 0 || ym < 0 || !dw || !offsets ||
      (n > 0 && (!x || !dy || !order)))
    return fail(MACE_ERR_BAD_ARG, "mace_species_linear_wgrad: bad arguments");
  if (unaligned(xs ? 1 : value_size(dtype), x) || unaligned(value_size(dtype), dy, dw) || unaligned(4, xs, order, offsets))
    return fail(MACE_ERR_BAD_ARG, "mace_species_linear_wgrad: an address is not a multiple of its values' size");
  int64_t need = 0;
  mace_species_linear_wgrad_workspace(n, d, G, K, M, &need);
  if (!ws || ws_bytes < need || (reinterpret_cast<uintptr_t>(ws) & 31) != 0)
    return fail(MACE_ERR_BAD_ARG, "mace_species_linear_wgrad: workspace too small or not 32-byte aligned");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int es = dtype == MACE_F32 ? 4 : 2, xe = xs ? 1 : es;
  SlParams p{};
  p.a = row_view(x, xn, xm, K, xe);
  p.b = row_view(dy, yn, ym, M, es);
  set_divisor(&p, d);
  p.a_scale = xs;
  p.ka_blocks = (K + MACE_CHECKPOINT_BLOCK - 1) / MACE_CHECKPOINT_BLOCK;
  p.out = dw;
  p.vst = vector_bytes(dw, (int64_t)M * es, 0, 0);
  p.part = static_cast<float*>(ws);
  p.order = order;
  p.offsets = offsets;
  p.n = n;
  p.d = d;
  p.G = G;
  p.K = K;
  p.N = M;
  p.alpha = alpha;
  wgrad_split(n, d, G, K, M, &p);
  if (n == 0) {
    MACE_CUDA_TRY(cudaMemsetAsync(dw, 0, (size_t)G * K * M * es, s));
    return MACE_OK;
  }
  p.spans = reinterpret_cast<int*>(static_cast<char*>(ws) + partial_bytes(p));
  const int grid = p.shares * p.n_ct * p.n_kt;
  const bool vec = aligned_rows(p.a, n, d, xe) && aligned_rows(p.b, n, d, es);
  auto go = [&](auto ta, auto t) {
    using TA = decltype(ta);
    using T = decltype(t);
    return vec ? launch_wgrad<TA, T, true>(p, grid, s) : launch_wgrad<TA, T, false>(p, grid, s);
  };
  int rc;
  if (xs)
    rc = dtype == MACE_F32 ? go(int8_t{}, float{}) : go(int8_t{}, bf16{});
  else if (dtype == MACE_F32)
    rc = go(float{}, float{});
  else  // bf16 in whole pieces: nothing to convert
    rc = vec ? launch_direct<true>(p, grid, s) : launch_wgrad<bf16, bf16, false>(p, grid, s);
  if (rc) return rc;
  const dim3 jg(G, 16 * (G > 16 ? 1 : p.NT / 32), std::min(p.n_ct * p.n_kt, 65535));  // (a grid's z; there may be one tile more)
  return launch("species_wgrad_join", dtype == MACE_F32 ? k_species_wgrad_join<float> : k_species_wgrad_join<bf16>, jg, 256,
                0, s, p);
}

extern "C" int mace_species_error_flag(int32_t* flag) {
  if (!flag) return fail(MACE_ERR_BAD_ARG, "mace_species_error_flag: null flag");
  MACE_CUDA_TRY(cudaDeviceSynchronize());
  MACE_CUDA_TRY(cudaMemcpyFromSymbol(flag, g_species_error, 4));
  const int zero = 0;
  MACE_CUDA_TRY(cudaMemcpyToSymbol(g_species_error, &zero, 4));
  return MACE_OK;
}
