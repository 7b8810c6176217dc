// Grouped-head attention, forward, on the tensor cores (16-bit inputs).
//
// One block owns 128 query rows of one event and head and walks the event's
// keys in tiles of kBN, twice resident on each SM so that one block's softmax
// runs beside the other's products:
//   warp 4   brings Q once and the K and V tiles by TMA;
//   warp 5   issues S = Q K^T into tensor memory, one tile ahead (two S
//            buffers), and O += P V from it;
//   warps 0-3, one thread a query row: reads S, keeps the running maximum and
//            sum, writes P back over S as 16-bit values (the A operand of the
//            second product), rescales O when the maximum has grown.
//
// Softmax in the base-2 domain: p = 2^(c s - c m), c = |scale| log2(e) (the
// sign of the scale is the product's own negate bit). O and l are rescaled
// only when the maximum has grown by more than 2^8 since the last rescale:
// p <= 2^8 then, exact in effect because the same m divides out at the end.
//
// P is rounded to the input type for the second product (u of its type, the
// one rounding besides the output's); l sums the unrounded fp32 values.

#include <cuda_runtime.h>

#include <atomic>

#include "fst_grouped_tc.cuh"

namespace fst {
namespace grouped {
namespace {

constexpr int kBM = 128;
constexpr int kBN = 64;
constexpr int kThreads = 192;
constexpr float kGrow = 8.f;  // log2 of the growth that forces a rescale

template <int Boxes, int Stages>
struct FwdSmem {
  alignas(1024) char q[Boxes * kBM * 128];
  alignas(1024) char k[Stages][Boxes * kBN * 128];
  alignas(1024) char v[Stages][Boxes * kBN * 128];
  uint64_t q_full, k_full[Stages], k_empty[Stages], v_full[Stages], v_empty[Stages];
  uint64_t s_full[2], p_ready[2], pv_done[2];  // of even and odd tiles
  uint32_t tmem;
};

template <typename T, int Boxes, int Stages>
__global__ void __launch_bounds__(kThreads, 2)
    fwd_kernel(const __grid_constant__ TileMaps maps, const FstGroupedForwardArgs a, int blocks) {
  using Smem = FwdSmem<Boxes, Stages>;
  extern __shared__ char raw[];
  Smem& sm = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  constexpr int kCols = 256;  // two S buffers (P over them) of kBN = 64, O from 128
  const FstGroupedProblem& p = a.prob;
  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (warp == 4 && lane == 0) {
    mbar_init(smem_addr(&sm.q_full), 1);
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
  __syncwarp();
  const BlockAt at = block_at(p, blocks);
  RowTile t;
  if (!find_tile<kBM>(p, at.id, p.causal, t)) return;
  const int D = p.head_dim;
  zero_dead_rows<T, kBM>(a.out, t, at.h, D, kThreads);
  if (t.i0 >= t.len) return;
  const int end = p.causal ? min(t.len, t.i0 + kBM) : t.len;
  const int tiles = (end + kBN - 1) / kBN;

  auto load = [&](int it, const CUtensorMap* map, char* dst, uint64_t* full) {
    const uint32_t bar = smem_addr(full);
    mbar_arrive_tx(bar, Boxes * kBN * 128);
    load_boxes<Boxes, kBN>(smem_addr(dst), map, bar, t.base + it * kBN, at.kh, t.ev);
  };
  if (warp == 4 && lane == 0) {
    // The first tiles set out before the others are ready for them.
    mbar_arrive_tx(smem_addr(&sm.q_full), Boxes * kBM * 128);
    load_boxes<Boxes, kBM>(smem_addr(sm.q), &maps.q, smem_addr(&sm.q_full), t.base + t.i0, at.h,
                           t.ev);
    for (int it = 0; it < Stages && it < tiles; ++it) {
      load(it, &maps.k, sm.k[it], &sm.k_full[it]);
      load(it, &maps.v, sm.v[it], &sm.v_full[it]);
    }
  }
  if (warp == 5) tmem_alloc<kCols>(smem_addr(&sm.tmem));
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem;
  const uint32_t tS = tmem, tO = tmem + 128;

  bool ok = true;
  if (warp == 4) {
    if (lane == 0) {
      for (int it = Stages; it < tiles; ++it) {
        const int s = it % Stages, last = (it / Stages - 1) & 1;
        ok = mbar_wait(smem_addr(&sm.k_empty[s]), last);
        if (!ok) break;
        load(it, &maps.k, sm.k[s], &sm.k_full[s]);
        ok = mbar_wait(smem_addr(&sm.v_empty[s]), last);
        if (!ok) break;
        load(it, &maps.v, sm.v[s], &sm.v_full[s]);
      }
    }
  } else if (warp == 5) {
    const uint32_t leader = elect_one();
    const int n = uniform(tiles), last = uniform(end), dim = uniform(D);
    const uint32_t s_mem = uniform(tS), o_mem = s_mem + 128;
    const uint32_t o_instr = instruction<T>((dim + 15) & ~15, true, false);
    auto keys = [&](int it) { return min(kBN, last - it * kBN); };
    // S of a tile. Its buffer may be overwritten: MMAs complete in order,
    // so the product that read P from it two tiles ago is done by then.
    auto logits = [&](int it) {
      const int s = it % Stages;
      if (!mbar_wait(smem_addr(&sm.k_full[s]), (it / Stages) & 1)) return false;
      product<T, Boxes, kBM, kBN>(s_mem + it % 2 * kBN, smem_addr(sm.q), smem_addr(sm.k[s]), dim,
                                 (keys(it) + 15) & ~15, p.scale < 0.f, leader);
      tc_commit(smem_addr(&sm.s_full[it % 2]), leader);
      tc_commit(smem_addr(&sm.k_empty[s]), leader);
      return true;
    };
    ok = mbar_wait(smem_addr(&sm.q_full), 0) && logits(0) && (n == 1 || logits(1));
    for (int it = 0; it < n && ok; ++it) {
      const int s = it % Stages;
      ok = mbar_wait(smem_addr(&sm.v_full[s]), (it / Stages) & 1) &&
           mbar_wait(smem_addr(&sm.p_ready[it % 2]), (it / 2) & 1);
      if (!ok) break;
      tc_fence_after();
      accumulate<kBN>(o_mem, s_mem + it % 2 * kBN, smem_addr(sm.v[s]), keys(it), o_instr, it > 0,
                     leader);
      tc_commit(smem_addr(&sm.pv_done[it % 2]), leader);
      tc_commit(smem_addr(&sm.v_empty[s]), leader);
      if (it + 2 < n) ok = logits(it + 2);
    }
  } else {
    const uint32_t quad = (uint32_t)(warp * 32) << 16;
    const int i = t.i0 + warp * 32 + lane;
    // Above 0, so that a masked -inf stays -inf under a scale of 0.
    const float c2 = fmaxf(fabsf(p.scale) * kLog2e, 1e-37f);
    float m = -INFINITY, l = 0.f;
    for (int it = 0; it < tiles; ++it) {
      const int j0 = it * kBN, nk = min(kBN, end - j0);
      // Keys j0 <= j < j0 + lim are seen; `edge` when some row sees fewer
      // than the tile's keys.
      const int lim = (p.causal ? min(i + 1, t.len) : t.len) - j0;
      const bool edge = j0 + kBN > t.len || (p.causal && j0 + kBN > t.i0 + 1);
      const uint32_t tSt = tS + quad + it % 2 * kBN;
      ok = mbar_wait(smem_addr(&sm.s_full[it % 2]), (it / 2) & 1);
      // O += P V of two tiles ago: long done, but waited for, so that the
      // wait on the last one below can only mean that one.
      if (ok && it >= 2) ok = mbar_wait(smem_addr(&sm.pv_done[it % 2]), (it / 2 - 1) & 1);
      if (!ok) break;
      tc_fence_after();
      float s[kBN / 32][32];
#pragma unroll
      for (int c = 0; c < kBN / 32; ++c)
        if (c * 32 < nk) tmem_ld32(s[c], tSt + c * 32);
      tmem_wait_ld();
      float mx = m;
#pragma unroll
      for (int c = 0; c < kBN / 32; ++c) {
        if (c * 32 >= nk) continue;
        pin(s[c]);
        if (edge) {
#pragma unroll
          for (int e = 0; e < 32; ++e) s[c][e] = c * 32 + e < lim ? s[c][e] : -INFINITY;
        }
        float part[4] = {mx, mx, mx, mx};
#pragma unroll
        for (int e = 0; e < 32; e += 8)
#pragma unroll
          for (int f = 0; f < 4; ++f)
            part[f] = max3(part[f], s[c][e + 2 * f], s[c][e + 2 * f + 1]);
        mx = max3(max3(part[0], part[1], part[2]), part[3], part[3]);
      }
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
          }
          ok = mbar_wait(smem_addr(&sm.pv_done[(it - 1) % 2]), ((it - 1) / 2) & 1);
          if (!ok) break;
          tc_fence_after();
#pragma unroll 1
          for (int d = 0; d < D; d += 16) tmem_scale16(tO + quad + d, keep);
        }
      }
      const float off = m == -INFINITY ? 0.f : m * c2;
      const pair_t scale2 = pair(c2, c2), off2 = pair(-off, -off);
      pair_t sums = pair(0.f, 0.f);
#pragma unroll
      for (int c = 0; c < kBN / 32; ++c) {
        if (c * 32 >= nk) continue;
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          float2 x = split(fma2(pair(s[c][e], s[c][e + 1]), scale2, off2));
          x = make_float2(ex2(x.x), ex2(x.y));
          sums = add2(sums, pair(x.x, x.y));
          w[e / 2] = Elem<T>::pack(x.x, x.y);
        }
        tmem_st16(tSt + c * 16, w);
      }
      const float2 halves = split(sums);
      const float sum = halves.x + halves.y;
      l += sum;
      if (nk & 15) {
        // Keys up to the next multiple of 16 have p = 0, but what V holds
        // there (another event's rows) must not be able to make 0 * NaN.
        const int st = it % Stages;
        ok = mbar_wait(smem_addr(&sm.v_full[st]), (it / Stages) & 1);
        if (!ok) break;
        zero_tile_rows<Boxes, kBN>(sm.v[st], nk, (nk + 15) & ~15, threadIdx.x, 128);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_addr(&sm.p_ready[it % 2]));
    }
    if (ok) ok = mbar_wait(smem_addr(&sm.pv_done[(tiles - 1) % 2]), ((tiles - 1) / 2) & 1);
    tc_fence_after();
    const bool live = i < t.len;
    store_row<T>(live ? row_ptr<T>(a.out, t, at.h, i) : nullptr, tO + quad, D,
                 ok ? 1.f / l : NAN);
    if (live) a.lse[stat_at(p, t, p.heads, at.h, i)] = ok ? (m * c2 + log2f(l)) / kLog2e : NAN;
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  if (warp == 5) tmem_free<kCols>(tmem);
}

template <typename T, int Boxes, int Stages>
int launch(const FstGroupedForwardArgs& a, cudaStream_t st) {
  const FstGroupedProblem& p = a.prob;
  static std::atomic<uint64_t> done{0};
  const auto kernel = fwd_kernel<T, Boxes, Stages>;
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
  if (a.prob.head_dim <= 64) return launch<T, 1, 3>(a, st);
  return launch<T, 2, 2>(a, st);
}

}  // namespace

bool tc_takes(const FstGroupedForwardArgs& a) {
  const FstGroupedProblem& p = a.prob;
  return tc_type(p) && on_grid(p, a.q, p.heads) && on_grid(p, a.out, p.heads) &&
         on_grid(p, a.k, p.kv_heads) && on_grid(p, a.v, p.kv_heads);
}

int tc_forward(const FstGroupedForwardArgs& a, cudaStream_t st) {
  if (a.prob.dtype == FST_BF16) return launch_t<__nv_bfloat16>(a, st);
  return launch_t<__half>(a, st);
}

}  // namespace grouped
}  // namespace fst
