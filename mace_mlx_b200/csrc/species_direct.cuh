// The species-indexed linear map and its weight gradient for bf16 rows of whole 16-byte pieces: nothing has to be
// converted, so every operand is copied by cp.async straight into its place for the tensor core (included by
// species_linear.cu, which holds the general kernel and the shared parts).
//
//   map:              A = 128 grouped rows x 64 channels, K-major (a row's 128 bytes per line);
//                     B = weights (K, N): N-major as they lie; transposed (N, K): K-major as they lie
//   weight gradient:  A = x and B = dy, 64 rows x 128 channels each, M- and N-major as they lie
//
// all in the 128-byte swizzled layout (piece j of line l at j ^ (l & 7)), from a ring of DR_NS steps of 64.
// Accumulation stays in TMEM over a whole tile (map) or SL_LONG steps (weight gradient; the truncation of each
// addition is 2^-24 of the sum, the result is rounded to 8 bits).  Roles of a CTA (16 warps, one CTA per SM):
//   warps 0-3   rows of x;  warps 4-7  map: weights (kept while the tiles share them) and the MMAs, zero rows;
//               weight gradient: rows of dy;  warps 8-15  epilogue (weight gradient: warp 8 issues the MMAs)
// 600 000 rows 128 -> 128: map 58 us (5.3 TB/s; 47 is what HBM needs), weight gradient with the join 61 (general kernel
// 135); 300 007 rows 96 -> 96 in 89 groups 32 and 36 (17.6): 8 to 14 us of each are the start of the pipeline, weights
// and the join, the rest copies and hand-over.  Waits are bounded as in species_linear.cu.
#pragma once

namespace mace {

namespace {

constexpr int DR_NS = 6;      // steps in the ring
constexpr int DR_LAG = 4;     // copies in flight before a step is handed on
constexpr uint32_t DR_TMEM = 256;  // two accumulators of 128 columns

template <bool WG>
struct Dr {
  static constexpr int A = 128 * 128;              // A of a step: 16 KB
  static constexpr int STEP = WG ? 2 * A : A;      // weight gradient: dy behind it
  static constexpr int NW = WG ? 0 : 4;            // weight slots of 64 x 128
  static constexpr int OFF_W = DR_NS * STEP;
  static constexpr int STG = 32 * 128;             // map: an epilogue warp's staging
  static constexpr int OFF_STG = OFF_W + NW * A;
  static constexpr int OFF_PRE = OFF_STG + (WG ? 0 : 8 * STG);
  static constexpr int OFF_BAR = OFF_PRE + Groups::INTS * 4;
  static constexpr int NBAR = 2 * DR_NS + 4 + 8 + 1;
  static constexpr int BYTES = OFF_BAR + NBAR * 8 + 16;
  static_assert(BYTES <= 232448, "shared memory of a CTA");
};

// Descriptor of an M- or N-major operand: 64-element blocks DR 8 KB apart, groups of 8 K-lines 1 KB apart
__device__ __forceinline__ uint64_t mn_desc(uint32_t addr) {
  uint64_t d = (uint64_t)((addr & 0x3FFFFu) >> 4);
  d |= (uint64_t)(8192 >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

__device__ __forceinline__ void mma_bf16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc), "r"(0u)
      : "memory");
}

template <bool WG>
__global__ void __launch_bounds__(SL_THREADS, 1) k_species_direct(const __grid_constant__ SlParams p) {
  using S = Dr<WG>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = tc::smem_u32(smem);
  const Groups q(smem + S::OFF_PRE);
  const int* const pre = q.pre;
  uint64_t* const bars = reinterpret_cast<uint64_t*>(smem + S::OFF_BAR);
  uint32_t* const tslot = reinterpret_cast<uint32_t*>(bars + S::NBAR);
  volatile int* const abort = reinterpret_cast<int*>(tslot + 1);
  auto bar = [&](int i) { return tc::smem_u32(bars + i); };
  auto FULL = [&](int s) { return bar(s); };
  auto FREE = [&](int s) { return bar(DR_NS + s); };
  auto D_FULL = [&](int s) { return bar(2 * DR_NS + s); };
  auto D_FREE = [&](int s) { return bar(2 * DR_NS + 2 + s); };
  auto W_FULL = [&](int s) { return bar(2 * DR_NS + 4 + s); };
  auto W_FREE = [&](int s) { return bar(2 * DR_NS + 8 + s); };
  const uint32_t DONE = bar(2 * DR_NS + 12);
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // known to be uniform
  const int NT = p.NT;

  if (base & 1023u) {  // the swizzled layout needs 1024-byte alignment
    if (tid == 0) atomicExch(&g_species_error, TC_ERR_ALIGN);
    return;
  }
  if (warp == 15) {  // while the others wait for the offsets
    if (lane == 0) {
      *abort = 0;
      for (int s = 0; s < DR_NS; ++s) {
        tc::mbar_init(FULL(s), WG ? 8 : 4);
        tc::mbar_init(FREE(s), 1);
      }
      for (int s = 0; s < 2; ++s) {
        tc::mbar_init(D_FULL(s), 1);
        tc::mbar_init(D_FREE(s), 8);
      }
      for (int s = 0; s < 4; ++s) {
        tc::mbar_init(W_FULL(s), 4);
        tc::mbar_init(W_FREE(s), 1);
      }
      tc::mbar_init(DONE, 1);
      tc::fence_barrier_init();
    }
    __syncwarp();
    tc::tmem_alloc(tc::smem_u32(tslot), DR_TMEM);
    tc::tmem_relinquish();
  }
  pdl_wait();  // nothing of the caller's is read or written before
  tc::fence_before_sync();
  const int tiles = WG ? p.n_ct * p.n_kt : 1;  // units and shares as in k_species_map and k_species_wgrad
  const int share = WG ? blockIdx.x / tiles : blockIdx.x;
  const int tile = WG ? blockIdx.x % tiles : 0;
  load_groups<SL_THREADS>(p, WG ? SL_KC : 128, WG ? 1 : p.n_ct, WG ? 0 : p.start, share, WG ? p.shares : gridDim.x, WG, q,
              reinterpret_cast<int64_t*>(smem));
  tc::fence_after_sync();
  const uint32_t tmem = *tslot;
  if (WG && blockIdx.x == 0) write_spans<SL_THREADS>(p, q);
  const int t0 = q.bounds[0], t1 = q.bounds[1];
  if (t0 >= t1) {
    if (!WG && warp >= 5 && warp < 8) zero_rows<bf16>(p);
    if (warp == 15) tc::tmem_dealloc(tmem, DR_TMEM);
    return;
  }
  const int wg_k0 = WG ? (tile / p.n_ct) * 128 : 0, wg_n0 = WG ? (tile % p.n_ct) * NT : 0;
  const int n_k = WG ? 1 : (p.K + SL_KC - 1) / SL_KC;  // steps of a tile
  const int steps = (t1 - t0) * n_k;
  const bool resident = n_k <= 4;  // map: the weights stay for the next row tile

  // copies of step i were issued in the i-th commit group of this thread: hand the step on once they have landed
  auto hand_on = [&](int i) {
    tc::fence_proxy_async();
    warp_arrive(FULL(i % DR_NS));
  };
  auto ring_loop = [&](auto&& copy) {
    bool ok = true;
#pragma unroll 1
    for (int i = 0; i < steps + DR_LAG && ok; ++i) {
      if (i < steps) {
        const int s = i % DR_NS;
        ok = i < DR_NS || wait_phase(FREE(s), (i / DR_NS - 1) & 1, abort);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        copy(base + s * S::STEP);
      }
      cp_commit();
      if (i >= DR_LAG) {
        cp_wait<DR_LAG>();
        hand_on(i - DR_LAG);
      }
    }
    cp_wait<0>();
  };

  if (warp < 4 || (WG && warp < 8)) {
    // ---------------- rows of x (or dy) ----------------
    const int w4 = warp & 3;
    if constexpr (!WG) {
      RowRef ref;
      Walk w;
      w.init(p, q, t0);
      uint32_t off[8];
      int k = 0;
      auto load_tile = [&]() {
        const Tile t(p, q, w);
        ref.load(p, t.at + w4 * 32 + lane, t.end);
      };
      load_tile();
      ring_loop([&](uint32_t dst) {
        if (k == 0) {
          // (a row outside the tile may hold anything: its TMEM lane is never stored)
          spread_rows(ref.valid(p) ? ref.pieces(p.a) : 0u, off);
          w.next(q, t1);
          if (w.t < t1) load_tile();
        }
        fetch_vec(dst + w4 * 4096, p.a.data, off, k * 128, p.a.width * 2);
        if (++k == n_k) k = 0;
      });
    } else {
      // 16 rows per warp and step; two lines of 64 channels per row.  Lane l: piece l % 16 of rows l / 16 + 2 i
      const RowView& v = warp < 4 ? p.a : p.b;
      const int at = (warp < 4 ? wg_k0 : wg_n0) * 2 + (lane & 15) * 16;  // byte within a row
      const bool past = at >= v.width * 2;
      const char* const src = past ? v.data : v.data + at;
      const uint32_t block = (warp < 4 ? 0 : S::A) + ((lane & 15) >> 3) * 8192 + w4 * 2048;
      const int j = lane & 7, half = lane >> 4;
      // the rows of two steps, loaded two steps ahead
      RowRef next[2];
      uint32_t now[2] = {NO_ROW, NO_ROW};
      Walk w;
      w.init(p, q, t0);
      auto load_pair = [&]() {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          next[u].m = -1;
          if (w.t < t1) {
            next[u].load(p, q.lo[w.g] * p.d + (w.t - pre[w.g]) * SL_KC + w4 * 16 + (lane & 15), q.hi[w.g] * p.d);
            w.next(q, t1);
          }
        }
      };
      next[0].node = next[1].node = -1;
      load_pair();
      int second = 0;
      ring_loop([&](uint32_t dst) {
        if (!second) {
#pragma unroll
          for (int u = 0; u < 2; ++u) now[u] = next[u].valid(p) ? next[u].pieces(v) : NO_ROW;
          load_pair();
        }
        const uint32_t mine = second ? now[1] : now[0];
        second ^= 1;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t o = __shfl_sync(0xffffffffu, mine, 2 * i + half);
          const bool none = o == NO_ROW;
          const int r = 2 * i + half;  // line within the warp's 16 (16 w4 is a multiple of 8)
          cp_async16_or_zero(dst + block + r * 128 + ((j ^ (r & 7)) << 4), none ? v.data : src + (uint64_t)o * 16,
                             past || none);
        }
      });
    }
  } else if (warp < 8) {
    // ---------------- map: weights and MMAs ----------------
    const int w4 = warp - 4;
    const uint32_t wbase = base + S::OFF_W;
    // step k of (g, ct) into slot s: transposed (N, K): line n, 64 K-values; else line k, two blocks of 64 columns
    auto fill = [&](int g, int ct, int k, int s) {
      const bf16* wt = static_cast<const bf16*>(p.w) + (int64_t)g * p.K * p.N;
      const uint32_t dst = wbase + s * S::A;
      const int r_end = p.transposed ? NT : SL_KC, pitch = p.transposed ? p.K : p.N;
      const int row0 = p.transposed ? ct * NT : k * SL_KC, rows = p.transposed ? p.N : p.K;
      if (p.transposed) {
        const int c = k * SL_KC + (lane & 7) * 8;
#pragma unroll 4
        for (int r = w4 * 4 + (lane >> 3); r < r_end; r += 16) {
          const bool in = row0 + r < rows && c < p.K;
          cp_async16_or_zero(dst + r * 128 + (((lane & 7) ^ (r & 7)) << 4), in ? wt + (int64_t)(row0 + r) * pitch + c : wt,
                             !in);
        }
      } else {
        const int c = ct * NT + (lane & 15) * 8;
#pragma unroll 4
        for (int r = w4 * 2 + (lane >> 4); r < r_end; r += 8) {
          const bool in = row0 + r < rows && c < p.N;
          cp_async16_or_zero(dst + ((lane & 15) >> 3) * 8192 + r * 128 + (((lane & 7) ^ (r & 7)) << 4),
                             in ? wt + (int64_t)(row0 + r) * pitch + c : wt, !in);
        }
      }
    };
    const uint32_t idesc = idesc_bf16(NT) | (p.transposed ? 0u : 1u << 16);  // B's major
    // step `it`, the first (and last) of its tile or not, with the weights of slot ws; use: as in k_species_map
    auto issue = [&](int it, int tile_no, bool first, bool last, int ws, int use, bool release) -> bool {
      const int s = it % DR_NS, ds = tile_no & 1;
      if (use >= 0 && !wait_phase(W_FULL(ws), use & 1, abort)) return false;
      if (!wait_phase(FULL(s), (it / DR_NS) & 1, abort)) return false;
      if (first && tile_no >= 2 && !wait_phase(D_FREE(ds), ((tile_no >> 1) - 1) & 1, abort)) return false;
      tc::fence_after_sync();
      const uint64_t ad = tc::sw128_desc(base + s * S::STEP);
      const uint32_t wa = wbase + ws * S::A;
      const uint64_t bd = p.transposed ? tc::sw128_desc(wa) : mn_desc(wa);
      const uint32_t hop = p.transposed ? 2 : 128;  // of 16 K-values, in 16 bytes
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) mma_bf16_ss(tmem + ds * 128, ad + ks * 2, bd + ks * hop, idesc, !first || ks > 0);
      tc::mma_commit(FREE(s));
      if (last) tc::mma_commit(D_FULL(ds));
      if (release) tc::mma_commit(W_FREE(ws));
      return true;
    };
    Walk w;
    w.init(p, q, t0);
    bool ok = true;
    int it = 0, tile_no = 0, fills = 0;
    while (w.t < t1 && ok) {
      const Tile t(p, q, w);
      if (resident) {
        // the tiles of this CTA that share the weights
        const int run = min(t.run, t1 - w.t);
        for (int k = 0; k < n_k && ok && fills > 0; ++k) ok = wait_phase(W_FREE(k), (fills - 1) & 1, abort);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        for (int k = 0; k < n_k; ++k) fill(w.g, t.ct, k, k);
        cp_commit();
        cp_wait<0>();
        tc::fence_proxy_async();
        for (int k = 0; k < n_k; ++k) warp_arrive(W_FULL(k));
        if (warp == 4 && elect_one())
          for (int i = 0; i < run && ok; ++i)
            for (int k = 0; k < n_k && ok; ++k)
              ok = issue(it + i * n_k + k, tile_no + i, k == 0, k + 1 == n_k, k, i == 0 ? fills : -1, i + 1 == run);
        it += run * n_k;
        tile_no += run;
        ++fills;
        w.t += run - 1;
      } else {
        for (int k = 0; k < n_k && ok; ++k, ++it, ++fills) {
          const int s = fills & 3, use = fills >> 2;
          ok = use == 0 || wait_phase(W_FREE(s), (use - 1) & 1, abort);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          fill(w.g, t.ct, k, s);
          cp_commit();
          cp_wait<0>();
          tc::fence_proxy_async();
          warp_arrive(W_FULL(s));
          if (warp == 4 && elect_one()) ok = issue(it, tile_no, k == 0, k + 1 == n_k, s, use, true);
          ok = __all_sync(0xffffffffu, ok);
        }
        ++tile_no;
      }
      ok = __all_sync(0xffffffffu, ok);
      w.next(q, t1);
    }
    if (warp == 4) {
      if (elect_one()) {
        tc::mma_commit(DONE);
        tc::mbar_wait(DONE, 0);
      }
      __syncwarp();
    } else {
      zero_rows<bf16>(p);
    }
  } else {
    // ---------------- epilogue ----------------
    const int quad = warp & 3, half = (warp - 8) >> 2;
    const int CW = NT / 2;  // columns of this warp: 16, 32, 48 or 64
    const uint32_t tq = tmem + ((uint32_t)(quad * 32) << 16) + half * CW;
    bool ok = true;
    Walk w;
    w.init(p, q, t0);
    if constexpr (!WG) {
      uint8_t* const stage = smem + S::OFF_STG + (warp - 8) * S::STG;
      RowRef ref;  // this lane's row of the next tile, loaded while the tile before it is stored
      int ct = 0;
      auto load_tile = [&]() {
        const Tile t(p, q, w);
        ref.load(p, t.at + quad * 32 + lane, t.end);
        ct = t.ct;
      };
      load_tile();
      for (int n = 0; w.t < t1; ++n) {
        const int s = n & 1;
        ok = __all_sync(0xffffffffu, wait_phase(D_FULL(s), (n >> 1) & 1, abort));
        if (!ok) break;
        tc::fence_after_sync();
        int row = lane;
        asm volatile("" : "+r"(row));  // (addresses made anew, as in copy_out)
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          uint32_t v[16];
          if (h * 16 < CW) tmem_ld16u(tq + s * 128 + h * 16, v);
          tc::tmem_wait_ld();
          if (h == 3) {
            tc::fence_before_sync();
            warp_arrive(D_FREE(s));
          }
          if (h * 16 < CW) {
            uint32_t o[8];
#pragma unroll
            for (int k = 0; k < 8; ++k)
              o[k] = pack_bf16(p.alpha * __uint_as_float(v[2 * k]), p.alpha * __uint_as_float(v[2 * k + 1]));
#pragma unroll
            for (int k = 0; k < 2; ++k)
              store_piece(stage + row * 128 + (((2 * h + k) ^ (row & 7)) << 4), o[4 * k], o[4 * k + 1], o[4 * k + 2],
                     o[4 * k + 3]);
          }
        }
        const RowRef here = ref;
        const int c0 = ct * NT + half * CW, left = min(p.N - c0, CW);
        w.next(q, t1);
        if (w.t < t1) load_tile();
        if (left > 0) copy_out<bf16>(p, stage, here, here.valid(p), c0, left);
        __syncwarp();
      }
    } else {
      // segments of up to SL_LONG steps of one group; warp 8 issues the next segment's MMAs before it takes this one's sum
      auto segment = [&](const Walk& x) { return min(min(SL_LONG, pre[x.g + 1] - x.t), t1 - x.t); };
      auto advance = [&](Walk& x, int n) {
        x.t += n - 1;
        x.next(q, t1);
      };
      const uint32_t idesc = idesc_bf16(NT) | (1u << 15) | (1u << 16);
      Walk m = w;  // the issuing side
      int mi = 0, ms = 0;
      auto issue = [&]() {
        if (warp != 8 || m.t >= t1) return;
        const int n = segment(m);
        if (elect_one()) {
          const int ds = ms & 1;
          if (ms >= 2) ok = wait_phase(D_FREE(ds), ((ms >> 1) - 1) & 1, abort);
          for (int i = 0; i < n && ok; ++i) {
            const int s = (mi + i) % DR_NS;
            ok = wait_phase(FULL(s), ((mi + i) / DR_NS) & 1, abort);
            if (!ok) break;
            tc::fence_after_sync();
            const uint64_t ad = mn_desc(base + s * S::STEP), bd = mn_desc(base + s * S::STEP + S::A);
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
              mma_bf16_ss(tmem + ds * 128, ad + ks * 128, bd + ks * 128, idesc, i > 0 || ks > 0);
            tc::mma_commit(FREE(s));
          }
          if (ok) tc::mma_commit(D_FULL(ds));
        }
        ok = __all_sync(0xffffffffu, ok);
        mi += n;
        ++ms;
        advance(m, n);
      };
      float acc[64];
      bool fresh = true;  // acc holds nothing yet
      issue();
      for (int n = 0; w.t < t1 && ok; ++n) {
        const int s = n & 1;
        issue();
        if (!ok) break;
        ok = __all_sync(0xffffffffu, wait_phase(D_FULL(s), (n >> 1) & 1, abort));
        if (!ok) break;
        tc::fence_after_sync();
        if (fresh) {
#pragma unroll
          for (int k = 0; k < 64; ++k) acc[k] = 0.f;
        }
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          uint32_t v[16];
          if (h * 16 < CW) tmem_ld16u(tq + s * 128 + h * 16, v);
          tc::tmem_wait_ld();
          if (h == 3) {
            tc::fence_before_sync();
            warp_arrive(D_FREE(s));
          }
#pragma unroll
          for (int k = 0; k < 16; k += 2) add2(acc[h * 16 + k], acc[h * 16 + k + 1], v[k], v[k + 1]);
        }
        fresh = false;
        const int len = segment(w);
        const bool group_ends = w.t + len == pre[w.g + 1];
        if (group_ends || w.t + len == t1) {
          finish_wgrad<bf16>(p, acc, w.g, group_ends && pre[w.g] >= t0, pre[w.g] > t0, tile, share, wg_k0, wg_n0,
                             quad * 32 + lane, half * CW, CW);
          fresh = true;
        }
        advance(w, len);
      }
      if (warp == 8) {
        if (elect_one()) {
          tc::mma_commit(DONE);
          tc::mbar_wait(DONE, 0);
        }
        __syncwarp();
      }
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  if (tid == 0 && *abort) atomicExch(&g_species_error, TC_ERR_TIMEOUT);
  if (warp == 15) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, DR_TMEM);
  }
}

template <bool WG>
int launch_direct(const SlParams& p, int grid, cudaStream_t s) {
  static bool attr_set[64] = {};
  return launch_big("species_direct", k_species_direct<WG>, attr_set, grid, SL_THREADS, Dr<WG>::BYTES, s, p);
}

}  // namespace

}  // namespace mace
