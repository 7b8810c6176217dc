// Grouped-head attention, backward, on the tensor cores (16-bit inputs): two
// kernels, each the only writer of its outputs, so the gradients need no
// atomics and are the same bits on every run.
//
// Row kernel (dq, and D_i = dO_i . o_i): a block owns 128 query rows of a head
// and walks the keys in tiles of 64:
//   S = Q K^T, dP = dO V^T  ->  dS = P (dP - D)  ->  dQ += dS K.
// Column kernel (dk, dv): a block owns 128 keys and walks the query rows, and
// the heads of the group, in tiles of 64, with the products transposed so
// that a thread owns a key:
//   S^T = K Q^T, dP^T = V dO^T  ->  dV += P^T dO, dK += dS^T Q.
// P and dS are written over S and dP in tensor memory as 16-bit values and are
// the A operands of the second products; each is rounded once to the type.
//
// P = 2^(c s - log2(e) lse) is recomputed in both. Splitting costs two of
// seven products and one exponential more than a single pass would take, and
// saves its fp32 additions into dq in memory, whose order would change with
// the schedule.

#include <cuda_runtime.h>

#include <atomic>

#include "fst_grouped_tc.cuh"

namespace fst {
namespace grouped {
namespace {

constexpr int kBM = 128;  // rows a block owns
constexpr int kBN = 64;   // rows of the other side per tile

// ---- dq ---------------------------------------------------------------------

template <int Boxes, int Stages>
struct RowSmem {
  alignas(1024) char q[Boxes * kBM * 128];
  alignas(1024) char g[Boxes * kBM * 128];
  alignas(1024) char k[Stages][Boxes * kBN * 128];
  alignas(1024) char v[Stages][Boxes * kBN * 128];
  uint64_t own_full, full[Stages], empty[Stages], s_full, ready, done;
  uint32_t tmem;
};

constexpr int kRowThreads = 192;

template <typename T, int Boxes, int Stages>
__global__ void __launch_bounds__(kRowThreads, 2)
    dq_kernel(const __grid_constant__ TileMaps maps, const FstGroupedBackwardArgs a, int blocks) {
  using Smem = RowSmem<Boxes, Stages>;
  extern __shared__ char raw[];
  Smem& sm = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  constexpr int kCols = 256;  // S (dS over it) 0, dP 64, dQ 128
  const FstGroupedProblem& p = a.prob;
  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const BlockAt at = block_at(p, blocks);
  RowTile t;
  if (!find_tile<kBM>(p, at.id, p.causal, t)) return;
  const int D = p.head_dim;
  zero_dead_rows<T, kBM>(a.dq, t, at.h, D, kRowThreads);
  if (t.i0 >= t.len) return;
  const int end = p.causal ? min(t.len, t.i0 + kBM) : t.len;
  const int tiles = (end + kBN - 1) / kBN;

  if (warp == 4) {
    tmem_alloc<kCols>(smem_addr(&sm.tmem));
  } else if (threadIdx.x == 0) {
    mbar_init(smem_addr(&sm.own_full), 1);
    for (int s = 0; s < Stages; ++s) {
      mbar_init(smem_addr(&sm.full[s]), 1);
      mbar_init(smem_addr(&sm.empty[s]), 1);
    }
    mbar_init(smem_addr(&sm.s_full), 1);
    mbar_init(smem_addr(&sm.ready), 4);
    mbar_init(smem_addr(&sm.done), 1);
    mbar_init_fence();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tS = sm.tmem, tP = tS + 64, tQ = tS + 128;

  bool ok = true;
  if (warp == 4) {
    if (lane == 0) {
      const uint32_t own = smem_addr(&sm.own_full);
      mbar_arrive_tx(own, 2 * Boxes * kBM * 128);
      load_boxes<Boxes, kBM>(smem_addr(sm.q), &maps.q, own, t.base + t.i0, at.h, t.ev);
      load_boxes<Boxes, kBM>(smem_addr(sm.g), &maps.g, own, t.base + t.i0, at.h, t.ev);
      for (int it = 0; it < tiles; ++it) {
        const int s = it % Stages, round = it / Stages;
        if (round) ok = mbar_wait(smem_addr(&sm.empty[s]), (round - 1) & 1);
        if (!ok) break;
        const uint32_t full = smem_addr(&sm.full[s]);
        mbar_arrive_tx(full, 2 * Boxes * kBN * 128);
        load_boxes<Boxes, kBN>(smem_addr(sm.k[s]), &maps.k, full, t.base + it * kBN, at.kh, t.ev);
        load_boxes<Boxes, kBN>(smem_addr(sm.v[s]), &maps.v, full, t.base + it * kBN, at.kh, t.ev);
      }
    }
  } else if (warp == 5) {
    const uint32_t leader = elect_one();
    const int n = uniform(tiles), last = uniform(end), dim = uniform(D);
    const uint32_t s_mem = uniform(tS);
    const uint32_t acc_instr = instruction<T>((dim + 15) & ~15, true, false);
    ok = mbar_wait(smem_addr(&sm.own_full), 0);
    for (int it = 0; it < n && ok; ++it) {
      const int s = it % Stages;
      const int keys = min(kBN, last - it * kBN), up = (keys + 15) & ~15;
      ok = mbar_wait(smem_addr(&sm.full[s]), (it / Stages) & 1);
      if (!ok) break;
      product<T, Boxes, kBM, kBN>(s_mem, smem_addr(sm.q), smem_addr(sm.k[s]), dim, up,
                                  p.scale < 0.f, leader);
      product<T, Boxes, kBM, kBN>(s_mem + 64, smem_addr(sm.g), smem_addr(sm.v[s]), dim, up, false,
                                  leader);
      tc_commit(smem_addr(&sm.s_full), leader);
      ok = mbar_wait(smem_addr(&sm.ready), it & 1);
      if (!ok) break;
      tc_fence_after();
      accumulate<kBN>(s_mem + 128, s_mem, smem_addr(sm.k[s]), keys, acc_instr, it > 0, leader);
      tc_commit(smem_addr(&sm.empty[s]), leader);
    }
    if (ok) tc_commit(smem_addr(&sm.done), leader);
  } else {
    const uint32_t quad = (uint32_t)(warp * 32) << 16;
    const int i = t.i0 + warp * 32 + lane;
    const bool live = i < t.len;
    const float c2 = fabsf(p.scale) * kLog2e;
    float lse2 = 0.f, delta = 0.f;
    if (live) {
      const T* o = row_ptr<T>(a.out, t, at.h, i);
      const T* g = row_ptr<T>(a.dout, t, at.h, i);
      for (int d = 0; d < D; d += 8) {
        const uint4 x = *(const uint4*)(o + d), y = *(const uint4*)(g + d);
        delta += Elem<T>::lo(x.x) * Elem<T>::lo(y.x) + Elem<T>::hi(x.x) * Elem<T>::hi(y.x);
        delta += Elem<T>::lo(x.y) * Elem<T>::lo(y.y) + Elem<T>::hi(x.y) * Elem<T>::hi(y.y);
        delta += Elem<T>::lo(x.z) * Elem<T>::lo(y.z) + Elem<T>::hi(x.z) * Elem<T>::hi(y.z);
        delta += Elem<T>::lo(x.w) * Elem<T>::lo(y.w) + Elem<T>::hi(x.w) * Elem<T>::hi(y.w);
      }
      const int64_t st = stat_at(p, t, p.heads, at.h, i);
      lse2 = a.lse[st] * kLog2e;
      a.delta[st] = delta;
    }
    const pair_t scale2 = pair(c2, c2), lse2n = pair(-lse2, -lse2), delta2n = pair(-delta, -delta);
    for (int it = 0; it < tiles; ++it) {
      const int j0 = it * kBN, nk = min(kBN, end - j0);
      const int lim = (p.causal ? min(i + 1, t.len) : t.len) - j0;
      const bool edge = j0 + kBN > t.len || (p.causal && j0 + kBN > t.i0 + 1);
      ok = mbar_wait(smem_addr(&sm.s_full), it & 1);
      if (!ok) break;
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < kBN / 32; ++c) {
        if (c * 32 >= nk) continue;
        float s[32], dp[32];
        tmem_ld32(s, tS + quad + c * 32);
        tmem_ld32(dp, tP + quad + c * 32);
        tmem_wait_ld();
        pin(s);
        pin(dp);
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          float2 x = split(fma2(pair(s[e], s[e + 1]), scale2, lse2n));
          x = split(mul2(pair(ex2(x.x), ex2(x.y)), add2(pair(dp[e], dp[e + 1]), delta2n)));
          s[e] = x.x;
          s[e + 1] = x.y;
        }
        if (edge) {
#pragma unroll
          for (int e = 0; e < 32; ++e) s[e] = c * 32 + e < lim ? s[e] : 0.f;
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) w[e] = Elem<T>::pack(s[2 * e], s[2 * e + 1]);
        tmem_st16(tS + quad + c * 16, w);
      }
      if (nk & 15)  // dS is 0 there, and must not meet another event's NaN
        zero_tile_rows<Boxes, kBN>(sm.k[it % Stages], nk, (nk + 15) & ~15, threadIdx.x, 128);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_addr(&sm.ready));
    }
    if (ok) ok = mbar_wait(smem_addr(&sm.done), 0);
    tc_fence_after();
    store_row<T>(live ? row_ptr<T>(a.dq, t, at.h, i) : nullptr, tQ + quad, D,
                 ok ? p.scale : NAN);
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  if (warp == 4) tmem_free<kCols>(tS);
}

// ---- dk, dv -----------------------------------------------------------------

// Groups: warpgroups of the block that turn S^T and dP^T into P^T and dS^T, on
// alternate tiles, each with its own pair of accumulators.
template <int Boxes, int Stages, int Groups>
struct ColSmem {
  alignas(1024) char k[Boxes * kBM * 128];
  alignas(1024) char v[Boxes * kBM * 128];
  alignas(1024) char q[Stages][Boxes * kBN * 128];
  alignas(1024) char g[Stages][Boxes * kBN * 128];
  alignas(16) float lse2n[Stages][kBN];   // -log2(e) lse of the query rows
  alignas(16) float deltan[Stages][kBN];  // -D
  uint64_t own_full, full[Stages], empty[Stages], s_full[Groups], ready[Groups], done;
  uint32_t tmem;
};

constexpr int col_threads(int groups) { return groups * 128 + 64; }

template <typename T, int Boxes, int Stages, int Groups>
__global__ void __launch_bounds__(col_threads(Groups), Groups == 1 ? 2 : 1)
    dkv_kernel(const __grid_constant__ TileMaps maps, const FstGroupedBackwardArgs a, int blocks) {
  using Smem = ColSmem<Boxes, Stages, Groups>;
  extern __shared__ char raw[];
  Smem& sm = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  constexpr int kThreads = col_threads(Groups);
  constexpr int kAcc = Boxes * 64;                    // columns of dV and of dK
  constexpr int kCols = Groups * 128 + 2 * kAcc;      // 256 or 512
  constexpr int kTma = Groups * 4, kMma = kTma + 1;   // warps
  const FstGroupedProblem& p = a.prob;
  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int kh = blockIdx.x / blocks, id = blockIdx.x - kh * blocks;
  const int group = p.heads / p.kv_heads;
  RowTile t;
  if (!find_tile<kBM>(p, id, false, t)) return;
  const int D = p.head_dim;
  zero_dead_rows<T, kBM>(a.dk, t, kh, D, kThreads);
  zero_dead_rows<T, kBM>(a.dv, t, kh, D, kThreads);
  if (t.i0 >= t.len) return;
  const int first = p.causal ? t.i0 : 0;                    // first query row
  const int per_head = (t.len - first + kBN - 1) / kBN;     // query tiles a head
  const int tiles = per_head * group;

  if (warp == kTma) {
    tmem_alloc<kCols>(smem_addr(&sm.tmem));
  } else if (threadIdx.x == 0) {
    mbar_init(smem_addr(&sm.own_full), 1);
    for (int s = 0; s < Stages; ++s) {
      mbar_init(smem_addr(&sm.full[s]), 2);
      mbar_init(smem_addr(&sm.empty[s]), 1);
    }
    for (int w = 0; w < Groups; ++w) {
      mbar_init(smem_addr(&sm.s_full[w]), 1);
      mbar_init(smem_addr(&sm.ready[w]), 4);
    }
    mbar_init(smem_addr(&sm.done), 1);
    mbar_init_fence();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // Per group S^T and dP^T of 64 columns, then dV, dK.
  const uint32_t tmem = sm.tmem, tV = tmem + Groups * 128, tK = tV + kAcc;

  bool ok = true;
  if (warp == kTma) {
    if (lane == 0) {
      const uint32_t own = smem_addr(&sm.own_full);
      mbar_arrive_tx(own, 2 * Boxes * kBM * 128);
      load_boxes<Boxes, kBM>(smem_addr(sm.k), &maps.k, own, t.base + t.i0, kh, t.ev);
      load_boxes<Boxes, kBM>(smem_addr(sm.v), &maps.v, own, t.base + t.i0, kh, t.ev);
    }
    int h = kh * group, q0 = first;
    for (int it = 0; it < tiles; ++it) {
      const int s = it % Stages, round = it / Stages;
      if (round) ok = mbar_wait(smem_addr(&sm.empty[s]), (round - 1) & 1);
      if (!__all_sync(0xffffffffu, ok)) break;
      const uint32_t full = smem_addr(&sm.full[s]);
      if (lane == 0) {
        mbar_arrive_tx(full, 2 * Boxes * kBN * 128);
        load_boxes<Boxes, kBN>(smem_addr(sm.q[s]), &maps.q, full, t.base + q0, h, t.ev);
        load_boxes<Boxes, kBN>(smem_addr(sm.g[s]), &maps.g, full, t.base + q0, h, t.ev);
      }
      const int64_t st = stat_at(p, t, p.heads, h, q0);
#pragma unroll
      for (int r = lane; r < kBN; r += 32) {
        const bool live = q0 + r < t.len;
        sm.lse2n[s][r] = live ? a.lse[st + r] * -kLog2e : 0.f;
        sm.deltan[s][r] = live ? -a.delta[st + r] : 0.f;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(full);
      q0 += kBN;
      if (q0 >= t.len) {
        q0 = first;
        ++h;
      }
    }
  } else if (warp == kMma) {
    const uint32_t leader = elect_one();
    const int n = uniform(tiles), each = uniform(per_head), rows = uniform(t.len - first);
    const int dim = uniform(D);
    const uint32_t mem = uniform(tmem), v_mem = mem + Groups * 128, k_mem = v_mem + kAcc;
    const uint32_t acc_instr = instruction<T>((dim + 15) & ~15, true, false);
    auto rows_of = [&](int it) { return min(kBN, rows - it % each * kBN); };
    // S^T and dP^T of a tile into its group's accumulators. The MMAs run in
    // order, so those that read the tile before from there are done.
    auto logits = [&](int it) {
      const int s = it % Stages, w = it % Groups, up = (rows_of(it) + 15) & ~15;
      if (!mbar_wait(smem_addr(&sm.full[s]), (it / Stages) & 1)) return false;
      product<T, Boxes, kBM, kBN>(mem + w * 128, smem_addr(sm.k), smem_addr(sm.q[s]), dim, up,
                                  p.scale < 0.f, leader);
      product<T, Boxes, kBM, kBN>(mem + w * 128 + 64, smem_addr(sm.v), smem_addr(sm.g[s]), dim,
                                  up, false, leader);
      tc_commit(smem_addr(&sm.s_full[w]), leader);
      return true;
    };
    ok = mbar_wait(smem_addr(&sm.own_full), 0);
    for (int it = 0; it < Groups && it < n && ok; ++it) ok = logits(it);
    for (int it = 0; it < n && ok; ++it) {
      const int s = it % Stages, w = it % Groups, q_rows = rows_of(it);
      ok = mbar_wait(smem_addr(&sm.ready[w]), (it / Groups) & 1);
      if (!ok) break;
      tc_fence_after();
      accumulate<kBN>(v_mem, mem + w * 128, smem_addr(sm.g[s]), q_rows, acc_instr, it > 0, leader);
      accumulate<kBN>(k_mem, mem + w * 128 + 64, smem_addr(sm.q[s]), q_rows, acc_instr, it > 0,
                      leader);
      tc_commit(smem_addr(&sm.empty[s]), leader);
      if (it + Groups < n) ok = logits(it + Groups);
    }
    if (ok) tc_commit(smem_addr(&sm.done), leader);
  } else {
    const int w = warp / 4;
    const uint32_t quad = (uint32_t)(warp % 4 * 32) << 16;
    const uint32_t tS = tmem + w * 128 + quad, tP = tS + 64;
    const int j = t.i0 + warp % 4 * 32 + lane;
    const float c2 = fabsf(p.scale) * kLog2e;
    const pair_t scale2 = pair(c2, c2);
    for (int it = w; it < tiles; it += Groups) {
      const int s = it % Stages;
      const int q0 = first + it % per_head * kBN, nq = min(kBN, t.len - q0);
      const bool edge = nq < kBN || (p.causal && q0 < t.i0 + kBM - 1);
      const int lo = p.causal ? j - q0 : 0;  // query columns lo <= c < nq see key j
      ok = mbar_wait(smem_addr(&sm.full[s]), (it / Stages) & 1) &&
           mbar_wait(smem_addr(&sm.s_full[w]), (it / Groups) & 1);
      if (!ok) break;
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < kBN / 32; ++c) {
        if (c * 32 >= nq) continue;
        float x[32], dp[32];
        tmem_ld32(x, tS + c * 32);
        tmem_ld32(dp, tP + c * 32);
        tmem_wait_ld();
        pin(x);
        pin(dp);
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          const ulonglong2 ls = *(const ulonglong2*)&sm.lse2n[s][c * 32 + e];
          const ulonglong2 de = *(const ulonglong2*)&sm.deltan[s][c * 32 + e];
#pragma unroll
          for (int f = 0; f < 4; f += 2) {
            float2 y = split(fma2(pair(x[e + f], x[e + f + 1]), scale2, f ? ls.y : ls.x));
            y.x = ex2(y.x);
            y.y = ex2(y.y);
            const float2 ds = split(mul2(
                pair(y.x, y.y), add2(pair(dp[e + f], dp[e + f + 1]), f ? de.y : de.x)));
            x[e + f] = y.x;
            x[e + f + 1] = y.y;
            dp[e + f] = ds.x;
            dp[e + f + 1] = ds.y;
          }
        }
        if (edge) {
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const bool seen = c * 32 + e >= lo && c * 32 + e < nq;
            x[e] = seen ? x[e] : 0.f;
            dp[e] = seen ? dp[e] : 0.f;
          }
        }
        uint32_t wp[16], wd[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          wp[e] = Elem<T>::pack(x[2 * e], x[2 * e + 1]);
          wd[e] = Elem<T>::pack(dp[2 * e], dp[2 * e + 1]);
        }
        tmem_st16(tS + c * 16, wp);
        tmem_st16(tP + c * 16, wd);
      }
      if (nq & 15) {
        zero_tile_rows<Boxes, kBN>(sm.q[s], nq, (nq + 15) & ~15, threadIdx.x & 127, 128);
        zero_tile_rows<Boxes, kBN>(sm.g[s], nq, (nq + 15) & ~15, threadIdx.x & 127, 128);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_addr(&sm.ready[w]));
    }
    if (ok) ok = mbar_wait(smem_addr(&sm.done), 0);
    tc_fence_after();
    // The groups share the epilogue: one of two stores dV, the other dK.
    const bool live = j < t.len;
    if (w == 0)
      store_row<T>(live ? row_ptr<T>(a.dv, t, kh, j) : nullptr, tV + quad, D, ok ? 1.f : NAN);
    if (w == Groups - 1)
      store_row<T>(live ? row_ptr<T>(a.dk, t, kh, j) : nullptr, tK + quad, D,
                   ok ? p.scale : NAN);
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  if (warp == kTma) tmem_free<kCols>(tmem);
}

template <typename K>
int prepare(K kernel, int bytes, std::atomic<uint64_t>& done) {
  const int e = allow_dynamic_smem((const void*)kernel, bytes, done);
  if (e) return api_fail(FST_ERR_CUDA, "shared memory: %s", cudaGetErrorString((cudaError_t)e));
  return FST_OK;
}

template <typename T, int Boxes, int RowStages, int ColStages, int Groups>
int launch(const FstGroupedBackwardArgs& a, cudaStream_t st) {
  const FstGroupedProblem& p = a.prob;
  static std::atomic<uint64_t> row_done{0}, col_done{0};
  const auto rows_k = dq_kernel<T, Boxes, RowStages>;
  const auto cols_k = dkv_kernel<T, Boxes, ColStages, Groups>;
  const int row_bytes = (int)sizeof(RowSmem<Boxes, RowStages>) + 1024;
  const int col_bytes = (int)sizeof(ColSmem<Boxes, ColStages, Groups>) + 1024;
  int rc = prepare(rows_k, row_bytes, row_done);
  if (!rc) rc = prepare(cols_k, col_bytes, col_done);
  const int64_t rows = p.packed ? p.total_rows : p.max_len, events = p.packed ? 1 : p.batch;
  const int D = p.head_dim;
  TileMaps r, c;  // 128 own rows, 64 of the other side
  if (!rc) rc = tc::make_rows_map(&r.q, a.q, D, rows, p.heads, events, kBM);
  if (!rc) rc = tc::make_rows_map(&r.g, a.dout, D, rows, p.heads, events, kBM);
  if (!rc) rc = tc::make_rows_map(&r.k, a.k, D, rows, p.kv_heads, events, kBN);
  if (!rc) rc = tc::make_rows_map(&r.v, a.v, D, rows, p.kv_heads, events, kBN);
  if (!rc) rc = tc::make_rows_map(&c.q, a.q, D, rows, p.heads, events, kBN);
  if (!rc) rc = tc::make_rows_map(&c.g, a.dout, D, rows, p.heads, events, kBN);
  if (!rc) rc = tc::make_rows_map(&c.k, a.k, D, rows, p.kv_heads, events, kBM);
  if (!rc) rc = tc::make_rows_map(&c.v, a.v, D, rows, p.kv_heads, events, kBM);
  if (rc) return rc;
  const int blocks = (int)list_blocks(p, kBM);
  rows_k<<<(unsigned)(blocks * p.heads), kRowThreads, row_bytes, st>>>(r, a, blocks);
  cols_k<<<(unsigned)(blocks * p.kv_heads), col_threads(Groups), col_bytes, st>>>(c, a, blocks);
  count_launch(2);
  return FST_OK;
}

template <typename T>
int launch_t(const FstGroupedBackwardArgs& a, cudaStream_t st) {
  // Two blocks an SM where dK and dV of 64 columns leave tensor memory for
  // them; else one block with two groups.
  if (a.prob.head_dim <= 64) return launch<T, 1, 3, 4, 1>(a, st);
  return launch<T, 2, 1, 4, 2>(a, st);
}

}  // namespace

bool tc_takes(const FstGroupedBackwardArgs& a) {
  const FstGroupedProblem& p = a.prob;
  return tc_type(p) && on_grid(p, a.q, p.heads) && on_grid(p, a.out, p.heads) &&
         on_grid(p, a.dout, p.heads) && on_grid(p, a.dq, p.heads) &&
         on_grid(p, a.k, p.kv_heads) && on_grid(p, a.v, p.kv_heads) &&
         on_grid(p, a.dk, p.kv_heads) && on_grid(p, a.dv, p.kv_heads);
}

int tc_backward(const FstGroupedBackwardArgs& a, cudaStream_t st) {
  if (a.prob.dtype == FST_BF16) return launch_t<__nv_bfloat16>(a, st);
  return launch_t<__half>(a, st);
}

}  // namespace grouped
}  // namespace fst
