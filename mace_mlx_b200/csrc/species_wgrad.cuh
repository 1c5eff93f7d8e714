// Weight gradient dW[g] = alpha sum over the rows of g of x^T dy, for rows that have to be converted (fp32, 8-bit
// checkpoints of x, bf16 rows of any alignment); included by species_linear.cu, which holds the map and the shared
// parts, and described there.
//
// A step is 64 rows: A = their 128 channels of x (a TMEM lane per channel), B = NT columns of dy.  600 000 fp32 rows
// 128 x 128 take 131 us with the join (94 is what HBM needs; 8-bit x 121, of 59, with bf16 dy 121, of 36; 64 x 64 108,
// of 47): the schedulers
// issue in 70 % of the cycles, masks and permutes of the split keep their pipe busy in 64 %, HBM is at 4.7 TB/s.  With
// four warps for each operand a step took as long as a warp needs from its rows in shared memory to their pieces in
// the operand (147, 127 and 131 us), so each operand has two teams of four warps with 32 rows of every step each, and
// the accumulators of all 128 columns fit four warps.  Roles of a CTA (24 warps, one CTA per SM):
//   warps 0-3, 4-7     operand A, first and second half of a step: rows by cp.async into a private ring of units of
//                      16 rows, split in registers, stored to TMEM (32 lanes each)
//   warps 8-11, 12-15  operand B likewise, into the step's 128B-swizzled K-major image
//   warps 16-19        epilogue
//   warp 20            MMAs (21-23 idle: registers are dealt out to four warps at a time)
// A thread is launched with 80 registers and goes on with 64 (teams), 184 (epilogue) or 40:
// 4 x 64 + 184 + 40 = 6 x 80.
#pragma once

namespace mace {

namespace {

constexpr int WG_THREADS = 24 * 32;
constexpr int WG_REGS = 80, WG_REGS_TEAM = 64, WG_REGS_EPI = 184, WG_REGS_MMA = 40;
static_assert(4 * WG_REGS_TEAM + WG_REGS_EPI + WG_REGS_MMA <= 6 * WG_REGS, "registers of a CTA");
constexpr int WG_UNIT = 16;  // rows of a ring unit

// A team's rows of the CTA's steps, one per lane and step.  Their atoms come from `order` by cp.async, three steps
// ahead, through a ring of each warp's own (a step is shorter than a load from HBM takes).
struct TeamRows {
  static constexpr int AHEAD = 3, SLOTS = 4;
  static constexpr int BYTES = SLOTS * 32 * 8;
  RowRef now;
  int t, g;          // next step to be loaded, its group
  int at, end, last; // this lane's place in the grouped list, where the group's end, and its units
  int slot;          // of the next step to be taken
  uint8_t* mine;     // this lane's entry of slot 0: the atom; its component is 128 bytes on
  __device__ __forceinline__ void enter(const SlParams& p, const Groups& q, int team) {
    end = q.hi[g] * p.d;
    last = q.pre[g + 1];
    at = q.lo[g] * p.d + (t - q.pre[g]) * SL_KC + team * 32 + (threadIdx.x & 31);
  }
  __device__ __forceinline__ void load(const SlParams& p, const Groups& q, int t1, int team, int to) {
    if (t >= t1) return;
    const int a = min(at, end - 1);
    int i = a, m = 0;
    if (p.d > 1) {
      i = __umulhi((uint32_t)a, p.div_mul) >> p.div_shift;
      m = a - i * p.d;
    }
    uint8_t* const entry = mine + to * 256;
    cp_async4(tc::smem_u32(entry), p.order + i, 4u);
    *reinterpret_cast<int*>(entry + 128) = at < end ? m : -1;
    at += SL_KC;
    if (++t == last && t < t1) {
      while (q.pre[g + 1] <= t) ++g;
      enter(p, q, team);
    }
  }
  __device__ __forceinline__ void init(const SlParams& p, const Groups& q, int t0, int t1, int team, uint8_t* ring) {
    mine = ring + (threadIdx.x & 31) * 4;
    slot = 0;
    Walk w;
    w.init(p, q, t0);
    t = t0;
    g = w.g;
    enter(p, q, team);
#pragma unroll 1
    for (int k = 0; k < AHEAD; ++k) load(p, q, t1, team, k);
    cp_commit();
    cp_wait<0>();
  }
  // (the copy of a step's rows is older than the last AHEAD units, so the ring's waits have covered it)
  __device__ __forceinline__ void step(const SlParams& p, const Groups& q, int t1, int team) {
    now.node = load_as<int>(mine + slot * 256);
    now.m = load_as<int>(mine + slot * 256 + 128);
    load(p, q, t1, team, (slot + AHEAD) & (SLOTS - 1));
    slot = (slot + 1) & (SLOTS - 1);
  }
};

template <typename TA, typename T, bool VEC>
struct Wg {
  static constexpr int PA = sizeof(TA) == 4 ? 3 : 1;
  static constexpr int PB = sizeof(TA) == 2 ? 1 : 3;
  static constexpr bool LONG = PA == 1 && PB == 1;  // sums of several steps (the result is rounded to 8 bits)
  static constexpr int SEG_A = 32 * (int)sizeof(TA), SEG_B = 32 * (int)sizeof(T);  // bytes of a row in a unit
  static constexpr bool ANY_A = !VEC && sizeof(TA) < 4, ANY_B = !VEC && sizeof(T) < 4;  // see fetch_unit
  static constexpr int PITCH_A = SEG_A + (ANY_A ? 16 : 0), PITCH_B = SEG_B + (ANY_B ? 16 : 0);
  static constexpr int UNIT_A = WG_UNIT * PITCH_A, UNIT_B = WG_UNIT * PITCH_B;
  static constexpr int NU_A = sizeof(TA) == 4 ? 3 : (sizeof(T) == 4 ? 5 : 6), NU_B = sizeof(TA) == 4 ? 3 : (sizeof(T) == 4 ? 4 : 6);
  static constexpr int OFF_A = 2 * PB * SL_IMG;  // after the images of two steps
  static constexpr int OFF_B = OFF_A + 8 * NU_A * UNIT_A;
  static constexpr int OFF_ROWS = OFF_B + 8 * NU_B * UNIT_B;  // a warp's rows of the next steps
  static constexpr int OFF_MIS = OFF_ROWS + 16 * TeamRows::BYTES;                      // per unit and row: misalignment
  static constexpr int OFF_SCALE = OFF_MIS + 8 * ((ANY_A ? NU_A : 0) + (ANY_B ? NU_B : 0)) * WG_UNIT;  // per B unit and row: A's scale
  static constexpr int OFF_PRE = OFF_SCALE + (sizeof(TA) == 1 ? 8 * NU_B * WG_UNIT * 4 : 0);
  static constexpr int OFF_BAR = OFF_PRE + Groups::INTS * 4;
  static constexpr int NBAR = 13;
  static constexpr int BYTES = OFF_BAR + NBAR * 8 + 16;
  static_assert(BYTES <= 232448 && OFF_MIS % 16 == 0 && OFF_SCALE % 16 == 0 && OFF_PRE % 8 == 0, "shared memory of a CTA");
  // the rows of the units fetched before the first wait come from TeamRows::init, and later waits cover later ones
  static_assert(NU_A <= 2 * TeamRows::AHEAD && NU_B <= 2 * TeamRows::AHEAD, "units in flight");
};

__device__ __forceinline__ void tmem_st8u(uint32_t a, const uint32_t* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(a), "r"(v[0]), "r"(v[1]),
               "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// 16 row segments of SEG bytes from byte `at` of their rows into a ring unit; the rows are those of lanes
// h * 16 .. h * 16 + 15 of `rows` (zeros for a row that does not exist or past its end).  Aligned rows (VEC) come in
// 16-byte pieces, other rows of 4-byte values value by value, and those of smaller ones as the 16-byte pieces that
// contain the segment, mis[r] saying where it starts in the first.
// (600 000 rows 97 x 61: fp32 158 us, 8-bit x 151; with the 4-byte values in pieces too 163 and 162.)
template <bool VEC>
struct UnitRows {
  uint32_t mine, have;  // this lane's row in 16 bytes (aligned), which rows exist
  uint64_t from;        // others: this lane's row, 0 for none
  __device__ __forceinline__ void take(const SlParams& p, const RowView& v, const RowRef& ref, int at) {
    const bool ok = ref.valid(p);
    have = __ballot_sync(0xffffffffu, ok);
    if constexpr (VEC) {
      mine = ok ? ref.pieces(v) : 0u;
    } else {
      from = ok ? reinterpret_cast<uint64_t>(v.data + ref.offset(v) + at) : 0;
    }
  }
};

template <int SEG, int PITCH, bool VEC>
__device__ __forceinline__ void fetch_unit(uint32_t dst, const RowView& v, const UnitRows<VEC>& rows, int h, int at,
                                           uint8_t* mis) {
  const int lane = threadIdx.x & 31, row_bytes = v.width * (SEG / 32);
  if constexpr (VEC) {
    constexpr int PPR = SEG / 16, RPI = 32 / PPR;  // pieces of a row, rows per instruction
    const int j = lane % PPR, r0 = lane / PPR;
    dst += r0 * PITCH + j * 16;
    if (rows.have == 0xffffffffu && at + SEG <= row_bytes) {  // the usual unit: nothing is left out
      const char* const src = v.data + at + 16 * j;
#pragma unroll
      for (int i = 0; i < WG_UNIT / RPI; ++i) {
        const uint32_t o = __shfl_sync(0xffffffffu, rows.mine, h * 16 + i * RPI + r0);
        cp_async16(dst + i * RPI * PITCH, src + (uint64_t)o * 16);
      }
    } else {
      const bool past = at + 16 * j >= row_bytes;
      const char* const src = past ? v.data : v.data + at + 16 * j;
#pragma unroll
      for (int i = 0; i < WG_UNIT / RPI; ++i) {
        const int r = h * 16 + i * RPI + r0;
        const uint32_t o = __shfl_sync(0xffffffffu, rows.mine, r);
        cp_async16_or_zero(dst + i * RPI * PITCH, src + (uint64_t)o * 16, past || !((rows.have >> r) & 1u));
      }
    }
  } else if constexpr (SEG == 128) {
    const uint32_t to = dst + lane * 4;
    if (rows.have == 0xffffffffu && at + SEG <= row_bytes) {
#pragma unroll
      for (int r = 0; r < WG_UNIT; ++r)
        cp_async4(to + r * PITCH, reinterpret_cast<const char*>(__shfl_sync(0xffffffffu, rows.from, h * 16 + r)) + lane * 4);
    } else {
#pragma unroll
      for (int r = 0; r < WG_UNIT; ++r) {
        const uint64_t f = __shfl_sync(0xffffffffu, rows.from, h * 16 + r);
        const bool in = f != 0 && at + lane * 4 < row_bytes;
        cp_async4(to + r * PITCH, in ? reinterpret_cast<const char*>(f) + lane * 4 : v.data, in ? 4u : 0u);
      }
    }
  } else {
    // lane l: piece l % PPR of rows l / PPR + i RPI, then the last piece of row l
    constexpr int PPR = SEG / 16, RPI = 32 / PPR;
    const char* const dummy = reinterpret_cast<const char*>(reinterpret_cast<uint64_t>(v.data) & ~(uint64_t)15);
    const int seg = max(min(row_bytes - at, SEG), 0);  // bytes of a row in this segment
    if ((lane >> 4) == h) mis[lane & 15] = (uint8_t)(rows.from & 15);
    // (the segment and 16 bytes more are inside the rows: every piece is whole)
    const bool inside = rows.have == 0xffffffffu && at + SEG + 16 <= row_bytes;
    auto copy = [&](uint64_t f, int r, int j) {
      const char* const src = reinterpret_cast<const char*>((f & ~(uint64_t)15) + 16 * j);
      if (inside) {
        cp_async16(dst + r * PITCH + j * 16, src);
      } else {
        const int left = (int)(f & 15) + seg - 16 * j;
        const uint32_t bytes = f == 0 || seg == 0 || left <= 0 ? 0u : (left < 16 ? (uint32_t)left : 16u);
        // (a copy of no bytes still names an aligned address)
        cp_async16(dst + r * PITCH + j * 16, bytes ? src : dummy, bytes);
      }
    };
#pragma unroll
    for (int i = 0; i < WG_UNIT / RPI; ++i) {
      const int r = i * RPI + lane / PPR;
      copy(__shfl_sync(0xffffffffu, rows.from, h * 16 + r), r, lane % PPR);
    }
    const uint64_t f = __shfl_sync(0xffffffffu, rows.from, h * 16 + (lane & 15));
    if (lane < WG_UNIT) copy(f, lane, PPR);
  }
}

// As redo_map: rows 32 quad .. of this share's results and partial tiles of matrix tile (k0, n0), by the warp that stored
// them.  The values of an 8-bit checkpoint are those that restoring gives.
template <typename TA, typename T>
__device__ __noinline__ void redo_wgrad(const SlParams& p, const Groups& q, int t0, int t1, int tile, int share, int k0,
                                        int n0, int quad) {
  constexpr int CB = 16;  // columns at a time
  const int lane = threadIdx.x & 31, kl = quad * 32 + lane, k = k0 + kl;
  __syncwarp();
  Walk w;
  w.init(p, q, t0);
#pragma unroll 1
  while (w.t < t1) {
    const int begin = q.pre[w.g], end = min(q.pre[w.g + 1], t1);
    const bool whole = begin >= t0 && q.pre[w.g + 1] <= t1;
    const int64_t first = (int64_t)q.lo[w.g] * p.d;
    const int a0 = (int)(first + (int64_t)(w.t - begin) * SL_KC);
    const int a1 = (int)min(first + (int64_t)(end - begin) * SL_KC, (int64_t)q.hi[w.g] * p.d);
    T* const out = static_cast<T*>(p.out) + ((int64_t)w.g * p.K + k) * p.N + n0;
    float* const part = p.part + ((((int64_t)tile * p.shares + share) * 2 + (begin > t0)) * 32 * p.NT + kl) * 4;
#pragma unroll 1
    for (int c = 0; c < min(p.NT, p.N - n0); c += CB) {
      unsigned left = 0;  // columns that are NaN
      if (k < p.K)
#pragma unroll
        for (int j = 0; j < CB; ++j)
          if (c + j < p.NT && n0 + c + j < p.N) {
            const float v = whole ? to_f32(out[c + j]) : part[(c + j) / 4 * 512 + (c + j) % 4];
            left |= (unsigned)(v != v) << j;
          }
      if (!__any_sync(0xffffffffu, left != 0)) continue;
      float sum[CB] = {};
      unsigned open = left;  // those whose sum is not NaN yet
#pragma unroll 1
      for (int a = a0; a < a1 && __any_sync(0xffffffffu, open != 0); a += 32) {
        RowRef ref;  // lane r: row a + r
        ref.load(p, a + lane, a1);
        const int valid = ref.valid(p);
#pragma unroll 2
        for (int r = 0; r < 32; ++r) {
          const int64_t node = __shfl_sync(0xffffffffu, ref.node, r), m = __shfl_sync(0xffffffffu, ref.m, r);
          if (!__shfl_sync(0xffffffffu, valid, r)) continue;
          const T* const dy = reinterpret_cast<const T*>(p.b.data + node * p.b.sn + m * p.b.sm) + n0 + c;
          float x = 0.f;
          if (k < p.K) x = to_f32(reinterpret_cast<const TA*>(p.a.data + node * p.a.sn + m * p.a.sm)[k]);
          if constexpr (sizeof(TA) == 1) x *= p.a_scale[(node * p.d + m) * p.ka_blocks + k0 / MACE_CHECKPOINT_BLOCK];
#pragma unroll
          for (int j = 0; j < CB; ++j)
            if (n0 + c + j < p.N) sum[j] = __fmaf_rn(x, to_f32(dy[j]), sum[j]);
        }
#pragma unroll
        for (int j = 0; j < CB; ++j)
          if (sum[j] != sum[j]) open &= ~(1u << j);
      }
#pragma unroll
      for (int j = 0; j < CB; ++j)
        if ((left >> j) & 1u) {
          if (whole)
            out[c + j] = from_f32<T>(p.alpha * sum[j]);
          else
            part[(c + j) / 4 * 512 + (c + j) % 4] = sum[j];
        }
    }
    w.t = end - 1;
    w.next(q, t1);
  }
}

template <typename TA, typename T, bool VEC>
__global__ void __launch_bounds__(WG_THREADS, 1) k_species_wgrad(const __grid_constant__ SlParams p) {
  using S = Wg<TA, T, VEC>;
  constexpr int PA = S::PA, PB = S::PB;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = tc::smem_u32(smem);
  const Groups q(smem + S::OFF_PRE);
  const int* const pre = q.pre;
  uint64_t* const bars = reinterpret_cast<uint64_t*>(smem + S::OFF_BAR);
  uint32_t* const tslot = reinterpret_cast<uint32_t*>(bars + S::NBAR);
  volatile int* const abort = reinterpret_cast<int*>(tslot + 1);
  volatile int* const odd = reinterpret_cast<int*>(tslot + 2);  // something that entered the sums is not finite
  auto bar = [&](int i) { return tc::smem_u32(bars + i); };
  auto A_FULL = [&](int s) { return bar(s); };
  auto A_FREE = [&](int s) { return bar(2 + s); };
  auto D_FULL = [&](int s) { return bar(4 + s); };
  auto D_FREE = [&](int s) { return bar(6 + s); };
  auto B_FULL = [&](int s) { return bar(8 + s); };
  auto B_FREE = [&](int s) { return bar(10 + s); };
  const uint32_t DONE = bar(12);
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // known to be uniform
  const int NT = p.NT;

  if (base & 1023u) {  // the images need 1024-byte alignment
    if (tid == 0) atomicExch(&g_species_error, TC_ERR_ALIGN);
    return;
  }
  if (warp == 20) {  // while the others wait for the offsets
    if (lane == 0) {
      *abort = *odd = 0;
      for (int s = 0; s < 2; ++s) {
        tc::mbar_init(A_FULL(s), 8);
        tc::mbar_init(A_FREE(s), 1);
        tc::mbar_init(D_FULL(s), 1);
        tc::mbar_init(D_FREE(s), 4);
        tc::mbar_init(B_FULL(s), NT / 16);  // warps of both teams
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
  // units are the steps; blockIdx.x = share * tiles + tile
  const int tiles = p.n_ct * p.n_kt, share = blockIdx.x / tiles, tile = blockIdx.x % tiles;
  load_groups<WG_THREADS>(p, SL_KC, 1, 0, share, p.shares, true, q, reinterpret_cast<int64_t*>(smem));
  tc::fence_after_sync();
  if (blockIdx.x == 0) write_spans<WG_THREADS>(p, q);
  const int t0 = q.bounds[0], t1 = q.bounds[1];
  if (t0 >= t1) {
    if (warp == 20) tc::tmem_dealloc(SL_D, SL_TMEM);
    return;
  }
  const int k0 = (tile / p.n_ct) * 128, n0 = (tile % p.n_ct) * NT;

  if (warp < 16) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(WG_REGS_TEAM));
    const int team = (warp >> 2) & 1, w8 = warp & 7, w4 = warp & 3;
    const int units = 2 * (t1 - t0);
    TeamRows rows;
    UnitRows<VEC> unit;
    int left = units, slot_f = 0, slot = 0;
    bool ok = true;
    if (warp < 8) {
      // ---------------- operand A: memory -> ring -> registers -> TMEM ----------------
      constexpr int NU = S::NU_A;
      constexpr bool ANY = S::ANY_A;
      const uint32_t ring = base + S::OFF_A + w8 * NU * S::UNIT_A;
      uint8_t* const mis = smem + S::OFF_MIS + w8 * NU * WG_UNIT;
      const uint32_t ta = SL_A + team * WG_UNIT + ((uint32_t)(w4 * 32) << 16);
      const int at = (k0 + w4 * 32) * (int)sizeof(TA);
      rows.init(p, q, t0, t1, team, smem + S::OFF_ROWS + warp * TeamRows::BYTES);
      auto fetch = [&]() {
        if (left > 0) {
          const int h = left & 1;  // half of the team's rows
          --left;
          if (h == 0) {
            rows.step(p, q, t1, team);
            unit.take(p, p.a, rows.now, at);
          }
          fetch_unit<S::SEG_A, S::PITCH_A, VEC>(ring + slot_f * S::UNIT_A, p.a, unit, h, at, mis + slot_f * WG_UNIT);
          slot_f = slot_f + 1 == NU ? 0 : slot_f + 1;
        }
        cp_commit();
      };
#pragma unroll 1
      for (int i = 1 - NU; i < units; ++i) {
        if (i >= 0) cp_wait<NU - 2>();
        __syncwarp();
        fetch();
        if (i < 0) continue;
        const uint8_t* const src = smem + S::OFF_A + (w8 * NU + slot) * S::UNIT_A + lane * (int)sizeof(TA);
        const uint8_t* const ms = mis + slot * WG_UNIT;
        slot = slot + 1 == NU ? 0 : slot + 1;
        const int it = i >> 1, half = i & 1, s = it & 1;
        if (!half) {
          ok = it < 2 || wait_phase(A_FREE(s), ((it >> 1) - 1) & 1, abort);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc::fence_after_sync();
        }
        // this lane's channel of 16 rows
        uint32_t out[PA][WG_UNIT / 2];
        const uint4 off = ANY ? load_as<uint4>(ms) : make_uint4(0, 0, 0, 0);
        const uint32_t skip[4] = {off.x, off.y, off.z, off.w};  // a byte per row
#pragma unroll
        for (int r = 0; r < WG_UNIT; r += 2) {
          uint32_t t[3];
          split2<PA>(load_f32<TA>(src + r * S::PITCH_A + (skip[r >> 2] >> (8 * (r & 3)) & 0xff)),
                     load_f32<TA>(src + (r + 1) * S::PITCH_A + (skip[r >> 2] >> (8 * (r & 3) + 8) & 0xff)), t);
#pragma unroll
          for (int a = 0; a < PA; ++a) out[a][r / 2] = t[a];
        }
#pragma unroll
        for (int a = 0; a < PA; ++a) tmem_st8u(ta + (s * PA + a) * 32 + half * (WG_UNIT / 2), out[a]);
        if (half) {
          tc::tmem_wait_st();
          tc::fence_before_sync();
          warp_arrive(A_FULL(s));
        }
      }
    } else if (w4 * 32 < NT) {
      // ---------------- operand B: 64-wide images, one column n per thread ----------------
      constexpr int NU = S::NU_B;
      constexpr bool ANY = S::ANY_B;
      const int n = w4 * 32 + lane;
      const uint32_t ring = base + S::OFF_B + w8 * NU * S::UNIT_B;
      uint8_t* const mis = smem + S::OFF_MIS + ((S::ANY_A ? 8 * S::NU_A : 0) + w8 * NU) * WG_UNIT;
      float* const sc = reinterpret_cast<float*>(smem + S::OFF_SCALE) + w8 * NU * WG_UNIT;
      uint8_t* const img = smem;
      const int at = (n0 + w4 * 32) * (int)sizeof(T);
      rows.init(p, q, t0, t1, team, smem + S::OFF_ROWS + warp * TeamRows::BYTES);
      auto fetch = [&]() {
        if (left > 0) {
          const int h = left & 1;
          --left;
          if (h == 0) {
            rows.step(p, q, t1, team);
            unit.take(p, p.b, rows.now, at);
          }
          fetch_unit<S::SEG_B, S::PITCH_B, VEC>(ring + slot_f * S::UNIT_B, p.b, unit, h, at, mis + slot_f * WG_UNIT);
          if constexpr (sizeof(TA) == 1) {
            if ((lane >> 4) == h) {
              const RowRef& ref = rows.now;
              const bool in = ref.valid(p);
              const float* src = in ? p.a_scale + ((int64_t)ref.node * p.d + ref.m) * p.ka_blocks + k0 / MACE_CHECKPOINT_BLOCK
                                    : p.a_scale;
              cp_async4(tc::smem_u32(sc + slot_f * WG_UNIT + (lane & 15)), src, in ? 4u : 0u);
            }
          }
          slot_f = slot_f + 1 == NU ? 0 : slot_f + 1;
        }
        cp_commit();
      };
#pragma unroll 1
      for (int i = 1 - NU; i < units; ++i) {
        if (i >= 0) cp_wait<NU - 2>();
        __syncwarp();
        fetch();
        if (i < 0) continue;
        const uint8_t* const src = smem + S::OFF_B + (w8 * NU + slot) * S::UNIT_B + lane * (int)sizeof(T);
        const uint8_t* const ms = mis + slot * WG_UNIT;
        const uint8_t* const ss = reinterpret_cast<const uint8_t*>(sc + slot * WG_UNIT);
        slot = slot + 1 == NU ? 0 : slot + 1;
        const int it = i >> 1, half = i & 1, s = it & 1;
        if (!half) {
          ok = it < 2 || wait_phase(B_FREE(s), ((it >> 1) - 1) & 1, abort);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
        }
#pragma unroll
        for (int h = 0; h < WG_UNIT / 8; ++h) {
          float v[8], scale[8];
          const uint2 off = ANY ? load_as<uint2>(ms + 8 * h) : make_uint2(0, 0);
          if constexpr (sizeof(TA) == 1) load_eight(ss + 32 * h, scale, float{});
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            v[j] = load_f32<T>(src + (8 * h + j) * S::PITCH_B + ((j < 4 ? off.x : off.y) >> (8 * (j & 3)) & 0xff));
            if constexpr (sizeof(TA) == 1) v[j] *= scale[j];
          }
          put_eight<PB>(img + s * (PB * SL_IMG), SL_IMG, n, team * 4 + half * 2 + h, v);
        }
        if (half) {
          tc::fence_proxy_async();
          warp_arrive(B_FULL(s));
        }
      }
    }
    cp_wait<0>();
  } else {
    // the steps of one sum, within a group
    auto sum_steps = [&](const Walk& x) { return S::LONG ? min(min(SL_LONG, pre[x.g + 1] - x.t), t1 - x.t) : 1; };
    auto advance = [&](Walk& x, int n) {
      x.t += n - 1;
      x.next(q, t1);
    };
    Walk w;
    w.init(p, q, t0);
    bool ok = true;
    if (warp >= 20) {
      // ---------------- MMAs, by one elected thread ----------------
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(WG_REGS_MMA));
      if (warp == 20 && elect_one()) {
        using PR = Products<PA, PB>;
        const uint32_t idesc = idesc_bf16(NT), bhi = (uint32_t)(tc::sw128_desc(base) >> 32);
        int it = 0;
        for (int sn = 0; w.t < t1 && ok; ++sn) {
          const int n = sum_steps(w);
          const uint32_t dcol = SL_D + (sn & 1) * 128;
          ok = sn < 2 || wait_phase(D_FREE(sn & 1), ((sn >> 1) - 1) & 1, abort);
          for (int i = 0; i < n && ok; ++i, ++it) {
            const int s = it & 1;
            ok = wait_phase(B_FULL(s), (it >> 1) & 1, abort) && wait_phase(A_FULL(s), (it >> 1) & 1, abort);
            if (!ok) break;
            tc::fence_after_sync();
            const uint32_t blo = (uint32_t)tc::sw128_desc(base + s * (PB * SL_IMG));
            // (the stage as a constant: little is left to compute)
            auto emit = [&](auto stage) {
              constexpr uint32_t st = decltype(stage)::value;
#pragma unroll
              for (int k = 0; k < PR::n; ++k)
#pragma unroll
                for (int ks = 0; ks < SL_KC / 16; ++ks)
                  mma_bf16_ta(dcol, SL_A + (st * PA + PR::a(k)) * 32 + ks * 8, blo + PR::b(k) * (SL_IMG / 16) + ks * 2,
                              bhi, idesc, i > 0 || k > 0 || ks > 0);
            };
            if (s)
              emit(std::integral_constant<uint32_t, 1>{});
            else
              emit(std::integral_constant<uint32_t, 0>{});
            tc::mma_commit(A_FREE(s));
            tc::mma_commit(B_FREE(s));
          }
          if (ok) tc::mma_commit(D_FULL(sn & 1));
          advance(w, n);
        }
        tc::mma_commit(DONE);  // every MMA issued is complete (bounded)
        tc::mbar_wait(DONE, 0);
      }
      __syncwarp();
    } else {
      // ---------------- epilogue ----------------
      asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(WG_REGS_EPI));
      const int quad = warp & 3;
      const uint32_t tq = SL_D + ((uint32_t)(quad * 32) << 16);
      float acc[128];
      bool fresh = true;  // acc holds nothing yet
      // NaN once a value of x or of dy was not finite: what it enters is a row of this lane, or a column of every lane, of
      // which each warp watches a quarter
      float probe = 0.f;
      for (int sn = 0; w.t < t1 && ok; ++sn) {
        const int s = sn & 1;
        ok = __all_sync(0xffffffffu, wait_phase(D_FULL(s), (sn >> 1) & 1, abort));
        if (!ok) break;
        tc::fence_after_sync();
        if (fresh) {
#pragma unroll
          for (int k = 0; k < 128; ++k) acc[k] = 0.f;
        }
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          uint32_t v[2][16];
#pragma unroll
          for (int k = 0; k < 2; ++k)
            if (h * 32 + k * 16 < NT) tmem_ld16u(tq + s * 128 + h * 32 + k * 16, v[k]);
          tc::tmem_wait_ld();
          if (h == 3) {
            tc::fence_before_sync();
            warp_arrive(D_FREE(s));
          }
#pragma unroll
          for (int k = 0; k < 32; k += 2)
            add2(acc[h * 32 + k], acc[h * 32 + k + 1], v[k >> 4][k & 15], v[k >> 4][(k & 15) + 1]);
        }
        fresh = false;
        const int len = sum_steps(w);
        const bool group_ends = w.t + len == pre[w.g + 1];
        if (group_ends || w.t + len == t1) {
          const bool whole = group_ends && pre[w.g] >= t0, inside = pre[w.g] > t0;
          if constexpr (PB == 3) {
            probe = __fmaf_rn(acc[0], 0.f, probe);
#pragma unroll
            for (int b = 0; b < 4; ++b)
              if (b == quad && b * 32 < NT) {
                float t[2] = {};
#pragma unroll
                for (int k = 0; k < 32; ++k) t[k & 1] = __fmaf_rn(acc[b * 32 + k], 0.f, t[k & 1]);
                probe += t[0] + t[1];
              }
          }
          finish_wgrad<T>(p, acc, w.g, whole, inside, tile, share, k0, n0, quad * 32 + lane, 0, min(NT, 64));
          if (NT > 64) finish_wgrad<T>(p, acc + 64, w.g, whole, inside, tile, share, k0, n0, quad * 32 + lane, 64, NT - 64);
          fresh = true;
        }
        advance(w, len);
      }
      if constexpr (PB == 3) {
        if (probe != 0.f) *odd = 1;
        tc::named_sync(1, 128);
        if (ok && *odd) redo_wgrad<TA, T>(p, q, t0, t1, tile, share, k0, n0, quad);
      }
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  if (tid == 0 && *abort) atomicExch(&g_species_error, TC_ERR_TIMEOUT);
  if (warp == 20) {
    tc::fence_after_sync();
    tc::tmem_dealloc(SL_D, SL_TMEM);
  }
}

}  // namespace

}  // namespace mace
