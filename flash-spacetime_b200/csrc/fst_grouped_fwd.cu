// Grouped-head attention, forward, on the tensor cores (16-bit inputs).
//
// An item is 128 query rows of one event and head; its keys come in tiles of
// kBN. A block works through many items (Feed), two blocks to an SM, so that
// one's softmax runs beside the other's products:
//   warp 4   feeds: looks items up, brings Q and the K and V tiles by TMA;
//   warp 5   issues S = Q K^T into tensor memory, one tile ahead (two S
//            buffers), and O += P V from it;
//   warps 0-3, one thread a query row: reads S, keeps the running maximum and
//            sum, writes P back over S as 16-bit values (the A operand of the
//            second product), rescales O when the maximum has grown.
//
// Measured, bf16, 8192 rows, 16 heads, not causal: 494 us at Dh = 128 (1113
// TFLOP/s; the 64-wide Q K^T reads 4 KB of Q for every 2 KB of K, and O and
// two S fill the 256 columns), 414 us at 64 and 392 us at 32, where the 2.6e12
// exponentials a second are 57 % of the unit's 16 a cycle and SM: the rest is
// the chain from one tile's S to its P (load 200 cycles, maximum 100, vote 90,
// exponentials 770, stores and barriers 200). Tiles whose keys all rows see
// run without masks (16384 causal of 64: 540 -> 470 us when that came in).
//
// Softmax in the base-2 domain: p = 2^(c s - c m), c = |scale| log2(e) (the
// sign of the scale is the product's own negate bit). O and l are rescaled
// only when the maximum has grown by more than 2^8 since the last rescale:
// p <= 2^8 then, exact in effect because the same m divides out at the end.
//
// P is rounded to the input type for the second product (u of its type, the
// one rounding besides the output's). O is divided by the sum of the rounded
// values, so the weights that made it sum to 1 and a common offset of v passes
// through unharmed: the backward takes D = dO . O from it, and an offset's
// share of an error there would not cancel against dP (dq of three keys with
// v of mean 8: error 23 times that of one rounding, now 1.1). lse, from which
// the backward forms P anew, is that of the unrounded fp32 sum.

#include <cuda_runtime.h>

#include <atomic>
#include <type_traits>

#include "fst_grouped_tc.cuh"

namespace fst {
namespace grouped {
namespace {

constexpr int kBM = 128;
constexpr int kBN = 64;
constexpr int kThreads = 192;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kGrow = 8.f;  // log2 of the growth that forces a rescale

template <int Boxes, int Stages>
struct FwdSmem {
  alignas(1024) char q[Boxes * kBM * 128];
  alignas(1024) char k[Stages][Boxes * kBN * 128];
  alignas(1024) char v[Stages][Boxes * kBN * 128];
  Ones ones;
  Feed feed;
  uint64_t q_full, q_empty, o_free;
  uint64_t k_full[Stages], k_empty[Stages], v_full[Stages], v_empty[Stages];
  uint64_t s_full[2], p_ready[2], pv_done[2];  // of even and odd tiles
  uint32_t tmem;
};

// Low: what rounding the output leaves over is kept too (training).
template <typename T, int Boxes, int Stages, bool Low>
__global__ void __launch_bounds__(kThreads, 2)
    fwd_kernel(const __grid_constant__ TileMaps maps, const FstGroupedForwardArgs a, int blocks) {
  using Smem = FwdSmem<Boxes, Stages>;
  extern __shared__ char raw[];
  Smem& sm = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  // Two S buffers (P over them) of kBN = 64, O from 128; up to Dh = 64 the sum
  // of the rounded P from 192: a product with 16 columns of ones, which the
  // tensor cores have time for (16384 causal of 64: 472 -> 478 us; summed by
  // the softmax warps, three more instructions a pair, 520). Above, O takes all
  // columns, and those warps sum (8192 x 16 of 128: 489 -> 496 us).
  constexpr int kCols = 256;
  constexpr bool kOnes = Boxes == 1;
  const FstGroupedProblem& p = a.prob;
  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int D = p.head_dim;
  if (warp == 4 && lane == 0) {
    feed_init(sm.feed, 5);
    mbar_init(smem_addr(&sm.q_full), 1);
    mbar_init(smem_addr(&sm.q_empty), 1);
    mbar_init(smem_addr(&sm.o_free), 4);
    for (int s = 0; s < Stages; ++s) {
      mbar_init(smem_addr(&sm.k_full[s]), 1);
      mbar_init(smem_addr(&sm.k_empty[s]), 1);
      mbar_init(smem_addr(&sm.v_full[s]), 1);
      mbar_init(smem_addr(&sm.v_empty[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_addr(&sm.s_full[b]), 1);
      mbar_init(smem_addr(&sm.p_ready[b]), 4);
      mbar_init(smem_addr(&sm.pv_done[b]), 1);
    }
    mbar_init_fence();
    prefetch_map(&maps.q);
    prefetch_map(&maps.k);
    prefetch_map(&maps.v);
  }
  if (kOnes && warp == 0) fill_ones<T>(sm.ones, lane);
  if (warp == 5) tmem_alloc<kCols>(smem_addr(&sm.tmem));
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem;
  const uint32_t tS = tmem, tO = tmem + 128;
  // Two blocks of an SM that begin together would ask for the exponentials, and
  // for the tensor cores, at the same time all along: the one whose columns are
  // the upper half of tensor memory starts half a tile later.
  if (tmem & 256) {
    const uint32_t start = (uint32_t)clock();
    while ((uint32_t)clock() - start < 600) {
    }
  }

  // Barriers and buffers go by the tile's number n in the block's life; `live`
  // counts its items that have tiles.
  bool ok = true;
  if (warp == 4) {
    int c = 0, n = 0, live = 0, most = 0, index = blockIdx.x;
    for (int round = 0; index >= 0 && ok; ++round) {
      const BlockAt at = block_at(p, blocks, index);
      Item item;
      item.h = at.h;
      item.kh = at.kh;
      if (find_tile<kBM>(p, at.id, p.causal, item.t)) {
        const RowTile& t = item.t;
        item.end = p.causal ? min(t.len, t.i0 + kBM) : t.len;
        item.tiles = t.i0 < t.len ? (item.end + kBN - 1) / kBN : 0;
        item.whole = min(item.tiles, (p.causal ? min(t.len, t.i0 + 1) : t.len) / kBN);
        item.dead = min(t.i0 + kBM, t.lim) > t.len;
        item.out_at = row_ptr<T>(a.out, t, item.h, t.i0) - (T*)a.out.data;
        item.stat_at = stat_at(p, t, p.heads, item.h, t.i0);
        ok = feed_put(sm.feed, c++, item, most, lane);
        if (item.tiles && ok) {
          if (lane == 0) {
            if (live) ok = wait_item(smem_addr(&sm.q_empty), (live - 1) & 1, most);
            const uint32_t q_full = smem_addr(&sm.q_full);
            if (ok) {
              mbar_arrive_tx(q_full, Boxes * kBM * 128);
              load_boxes<Boxes, kBM>(smem_addr(sm.q), &maps.q, q_full, t.base + t.i0, item.h,
                                     t.ev);
            }
            for (int it = 0; it < item.tiles && ok; ++it) {
              const int s = (n + it) % Stages, round_of = (n + it) / Stages;
              auto load = [&](const CUtensorMap* map, char* dst, uint64_t* full, uint64_t* empty) {
                if (round_of && !mbar_wait(smem_addr(empty), (round_of - 1) & 1)) return false;
                const uint32_t bar = smem_addr(full);
                mbar_arrive_tx(bar, Boxes * kBN * 128);
                load_boxes<Boxes, kBN>(smem_addr(dst), map, bar, t.base + it * kBN, item.kh, t.ev);
                return true;
              };
              ok = load(&maps.k, sm.k[s], &sm.k_full[s], &sm.k_empty[s]) &&
                   load(&maps.v, sm.v[s], &sm.v_full[s], &sm.v_empty[s]);
            }
          }
          n += item.tiles;
          ++live;
          most = max(most, item.tiles);
          ok = __shfl_sync(0xffffffffu, ok, 0);
        }
      }
      // Asked for only now, with the item's last loads under way, so that no
      // block holds work that another has time for. After a wait that ran out,
      // not at all: what is asked for would be lost, its rows left as they were.
      if (!ok) break;
      if (lane == 0) feed_ask(sm.feed);
      __syncwarp();
      index = feed_answer(sm.feed, round);
    }
    Item last{};
    last.tiles = -1;
    feed_put(sm.feed, c, last, most, lane);
  } else if (warp == 5) {
    const uint32_t leader = elect_one();
    const int dim = uniform(D);
    const uint32_t s_mem = uniform(tS), o_mem = s_mem + 128;
    const uint32_t o_instr = instruction<T>((dim + 15) & ~15, true, false);
    Item item;
    for (int c = 0, n = 0, live = 0; ok && feed_take(sm.feed, c, item, lane); ++c) {
      const int tiles = uniform(item.tiles);
      if (!tiles) continue;
      const int last = uniform(item.end);
      auto keys = [&](int it) { return min(kBN, last - it * kBN); };
      // S of a tile. Its buffer may be overwritten: MMAs complete in order,
      // so the product that read P from it two tiles ago is done by then.
      auto logits = [&](int it) {
        const int g = n + it, s = g % Stages;
        if (!mbar_wait(smem_addr(&sm.k_full[s]), (g / Stages) & 1)) return false;
        product<T, Boxes, kBM, kBN>(s_mem + g % 2 * kBN, smem_addr(sm.q), smem_addr(sm.k[s]), dim,
                                    (keys(it) + 15) & ~15, p.scale < 0.f, leader);
        tc_commit(smem_addr(&sm.s_full[g % 2]), leader);
        tc_commit(smem_addr(&sm.k_empty[s]), leader);
        if (it + 1 == tiles) tc_commit(smem_addr(&sm.q_empty), leader);
        return true;
      };
      ok = mbar_wait(smem_addr(&sm.q_full), live & 1) && logits(0) && (tiles == 1 || logits(1));
      for (int it = 0; it < tiles && ok; ++it) {
        const int g = n + it, s = g % Stages;
        // The first product writes over O: the item before has read it.
        if (it == 0 && live) ok = mbar_wait(smem_addr(&sm.o_free), (live - 1) & 1);
        ok = ok && mbar_wait(smem_addr(&sm.v_full[s]), (g / Stages) & 1) &&
             mbar_wait(smem_addr(&sm.p_ready[g % 2]), (g / 2) & 1);
        if (!ok) break;
        tc_fence_after();
        accumulate<kBN>(o_mem, s_mem + g % 2 * kBN, smem_addr(sm.v[s]), keys(it), o_instr, it > 0,
                        leader);
        if (kOnes)
          row_sums<T, kBN>(o_mem + 64, s_mem + g % 2 * kBN, smem_addr(&sm.ones), keys(it), it > 0,
                           leader);
        tc_commit(smem_addr(&sm.pv_done[g % 2]), leader);
        tc_commit(smem_addr(&sm.v_empty[s]), leader);
        if (it + 2 < tiles) ok = logits(it + 2);
      }
      n += tiles;
      ++live;
    }
  } else {
    const uint32_t quad = (uint32_t)(warp * 32) << 16;
    // Above 0, so that a masked -inf stays -inf under a scale of 0.
    const float c2 = fmaxf(fabsf(p.scale) * kLog2e, 1e-37f);
    const pair_t scale2 = pair(c2, c2);
    Item item;
    for (int c = 0, n = 0; ok && feed_take(sm.feed, c, item, lane); ++c) {
      const RowTile& t = item.t;
      if (item.dead) zero_dead_rows<T, kBM>(a.out, t, item.h, D, 128);
      if (!item.tiles) continue;
      const int end = item.end;
      const int i = t.i0 + warp * 32 + lane;
      float m = -INFINITY, l = 0.f, l_used = 0.f;  // l_used: of the rounded P, if kOnes is not
      // One tile. `Whole`: every row of the block sees all its keys.
      auto tile = [&](auto whole, int it) {
        constexpr bool Whole = decltype(whole)::value;
        const int j0 = it * kBN, nk = Whole ? kBN : min(kBN, end - j0);
        const uint32_t tSt = tS + quad + n % 2 * kBN;
        if (!mbar_wait(smem_addr(&sm.s_full[n % 2]), (n / 2) & 1)) return false;
        tc_fence_after();
        float s[2][32];
        tmem_ld32(s[0], tSt);
        if (Whole || nk > 32) tmem_ld32(s[1], tSt + 32);
        tmem_wait_ld();
        pin(s[0]);
        pin(s[1]);
        if (!Whole) {
          // Keys below lim are seen; the warp's first row sees fewest.
          const int lim = (p.causal ? min(i + 1, t.len) : t.len) - j0, fewest = uniform(lim);
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            if (c * 32 + 32 <= fewest) continue;
#pragma unroll
            for (int e = 0; e < 32; ++e) s[c][e] = c * 32 + e < lim ? s[c][e] : -INFINITY;
          }
        }
        float part[8];
#pragma unroll
        for (int f = 0; f < 8; ++f) part[f] = max3(m, s[0][f], s[1][f]);
#pragma unroll
        for (int e = 8; e < 32; e += 8)
#pragma unroll
          for (int f = 0; f < 8; ++f) part[f] = max3(part[f], s[0][e + f], s[1][e + f]);
        const float mx = max3(max3(part[0], part[1], part[2]), max3(part[3], part[4], part[5]),
                              max3(part[6], part[7], part[7]));
        // First tile: O is written, not added to, so m may move freely.
        if (it == 0) {
          m = mx;
        } else {
          // (True for a NaN too, which then reaches O and l.)
          const bool grow = !((mx - m) * c2 <= kGrow) && mx != m;
          if (__any_sync(0xffffffffu, grow)) {
            const float keep = grow ? ex2((m - mx) * c2) : 1.f;
            if (grow) {
              m = mx;
              l *= keep;
              l_used *= keep;
            }
            if (!mbar_wait(smem_addr(&sm.pv_done[(n - 1) % 2]), ((n - 1) / 2) & 1)) return false;
            tc_fence_after();
#pragma unroll 1
            for (int d = 0; d < D; d += 16) tmem_scale16(tO + quad + d, keep);
            if (kOnes) tmem_scale16(tO + quad + 64, keep);
          }
        }
        const float off = m == -INFINITY ? 0.f : m * c2;
        const pair_t off2 = pair(-off, -off);
        pair_t sums = pair(0.f, 0.f), used = sums;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if (!Whole && c * 32 >= nk) continue;
          uint32_t w[16];
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            float2 x = split(fma2(pair(s[c][e], s[c][e + 1]), scale2, off2));
            x = make_float2(ex2(x.x), ex2(x.y));
            sums = add2(sums, pair(x.x, x.y));
            w[e / 2] = Elem<T>::pack(x.x, x.y);
            if (!kOnes) used = add2(used, pair(Elem<T>::lo(w[e / 2]), Elem<T>::hi(w[e / 2])));
          }
          tmem_st16(tSt + c * 16, w);
        }
        const float2 halves = split(sums);
        l += halves.x + halves.y;
        const float2 used_halves = split(used);
        l_used += used_halves.x + used_halves.y;
        if (!Whole && (nk & 15)) {
          // Keys up to the next multiple of 16 have p = 0, but what V holds
          // there (another event's rows) must not be able to make 0 * NaN.
          const int st = n % Stages;
          if (!mbar_wait(smem_addr(&sm.v_full[st]), (n / Stages) & 1)) return false;
          zero_tile_rows<Boxes, kBN>(sm.v[st], nk, (nk + 15) & ~15, threadIdx.x, 128);
        }
        // O += P V of two tiles ago: long done, but waited for on every tile,
        // so that the wait before a rescale can only mean the tile before.
        if (n >= 2 && !mbar_wait(smem_addr(&sm.pv_done[n % 2]), (n / 2 - 1) & 1)) return false;
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_addr(&sm.p_ready[n % 2]));
        ++n;
        return true;
      };
      int it = 0;
      for (; it < item.whole && ok; ++it) ok = tile(std::true_type(), it);
      for (; it < item.tiles && ok; ++it) ok = tile(std::false_type(), it);
      // All but the output itself, while the last product runs.
      const bool seen = i < t.len;
      const int row = i - t.i0;
      if (seen) a.lse[item.stat_at + row] = ok ? (m * c2 + log2f(l)) * kLn2 : NAN;
      T* out = seen ? (T*)a.out.data + item.out_at + row * a.out.row_stride : nullptr;
      if (ok) ok = mbar_wait(smem_addr(&sm.pv_done[(n - 1) % 2]), ((n - 1) / 2) & 1);
      tc_fence_after();
      if (kOnes) {
        l_used = tmem_ld1(tO + quad + 64);
        tmem_wait_ld();
        pin(l_used);
      }
      const float f = ok ? 1.f / l_used : NAN;
      T* low = Low && seen ? row_ptr<T>(a.out_low, t, item.h, i) : nullptr;
      if (Low && Boxes == 1) {
        store_row<T, false, true>(out, tO + quad, D, f, low);
      } else {
        // Two passes over a wide row: one would cost the main loop registers.
        store_row<T>(out, tO + quad, D, f);
        if (Low) store_row<T, true>(low, tO + quad, D, f);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_addr(&sm.o_free));
    }
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  if (warp == 5) tmem_free<kCols>(tmem);
}

template <typename T, int Boxes, int Stages, bool Low>
int launch(const FstGroupedForwardArgs& a, cudaStream_t st) {
  const FstGroupedProblem& p = a.prob;
  static std::atomic<uint64_t> done{0};
  const auto kernel = fwd_kernel<T, Boxes, Stages, Low>;
  const int bytes = (int)sizeof(FwdSmem<Boxes, Stages>) + 1024;
  const int e = allow_dynamic_smem((const void*)kernel, bytes, done);
  if (e) return api_fail(FST_ERR_CUDA, "shared memory: %s", cudaGetErrorString((cudaError_t)e));
  const int64_t rows = p.packed ? p.total_rows : p.max_len, events = p.packed ? 1 : p.batch;
  TileMaps maps;
  int rc = tc::make_rows_map(&maps.q, a.q, p.head_dim, rows, p.heads, events, kBM);
  if (!rc) rc = tc::make_rows_map(&maps.k, a.k, p.head_dim, rows, p.kv_heads, events, kBN);
  if (!rc) rc = tc::make_rows_map(&maps.v, a.v, p.head_dim, rows, p.kv_heads, events, kBN);
  if (rc) return rc;
  maps.g = maps.q;
  const int blocks = (int)list_blocks(p, kBM);
  kernel<<<(unsigned)(blocks * p.heads), kThreads, bytes, st>>>(maps, a, blocks);
  count_launch();
  return FST_OK;
}

template <typename T>
int launch_t(const FstGroupedForwardArgs& a, cudaStream_t st) {
  const bool low = a.out_low.data != nullptr;
  if (a.prob.head_dim <= 64) return low ? launch<T, 1, 3, true>(a, st) : launch<T, 1, 3, false>(a, st);
  return low ? launch<T, 2, 2, true>(a, st) : launch<T, 2, 2, false>(a, st);
}

}  // namespace

bool tc_takes(const FstGroupedForwardArgs& a) {
  const FstGroupedProblem& p = a.prob;
  return tc_type(p) && on_grid(p, a.q, p.heads) && on_grid(p, a.out, p.heads) &&
         (!a.out_low.data || on_grid(p, a.out_low, p.heads)) &&
         on_grid(p, a.k, p.kv_heads) && on_grid(p, a.v, p.kv_heads);
}

int tc_forward(const FstGroupedForwardArgs& a, cudaStream_t st) {
  if (a.prob.dtype == FST_BF16) return launch_t<__nv_bfloat16>(a, st);
  return launch_t<__half>(a, st);
}

}  // namespace grouped
}  // namespace fst
