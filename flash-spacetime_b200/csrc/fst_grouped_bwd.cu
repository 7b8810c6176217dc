// Grouped-head attention, backward, on the tensor cores (16-bit inputs): two
// kernels, each the only writer of its outputs, so the gradients need no
// atomics and are the same bits on every run.
//
// Row kernel (dq, and D_i = dO_i . o_i): a block owns 128 query rows of a head
// and walks the keys:
//   S = Q K^T, dP = dO V^T  ->  dS = P (dP - D)  ->  dQ += dS K.
// Column kernel (dk, dv): a block owns 128 keys and walks the query rows, and
// the heads of the group, with the products transposed so that a thread owns
// a key:
//   S^T = K Q^T, dP^T = V dO^T  ->  dV += P^T dO, dK += dS^T Q.
// P and dS are written over S and dP in tensor memory as 16-bit values and are
// the A operands of the second products; each is rounded once to the type.
//
// P = 2^(c s - log2(e) lse) is recomputed in both. Splitting costs two of
// seven products and one exponential more than a single pass would take, and
// saves its fp32 additions into dq in memory, whose order would change with
// the schedule.
//
// A tile goes through the tensor cores in two halves, so that they and the
// exponentials work at the same time on one pair of accumulators:
//   rows:     S of the next tile | dS of this one;  dQ, next dP | next P
//   columns:  dV, next S         | dS of this one;  dK, next dP | next P
// fp16 ends at 6e-5 below, where dS of a long event lies (P is 1 / n, and dO is
// small under a mean over many rows). So fp16 calls carry powers of two in P
// and dS, folded into the exponent and the statistics at no cost a pair, and
// taken back when the results are stored: dS of row i by the largest that
// |dS_ij| <= 2 Dh max|dO_i| max|v_j| keeps finite in the row kernel, by one of
// the event and key head in the column kernel, P of dV by 2^14. A short launch
// before the two finds the maxima (16384 causal, 8 of 64: backward 1290 -> 1304
// us). Error of dq and dk over that of one rounding, 4096 keys, Dh = 64, dO of
// 1, 1e-2, 1e-3: 1.4, 1.4, 1.1; without 1.4, 2.8, 8.1.
//
// W warpgroups share a tile of 64 W rows of the other side, 64 columns each.
// Up to Dh = 64 one group and 256 columns of tensor memory: two blocks an SM.
// Above, dV and dK (or dQ) need twice the columns; two groups and one block,
// whose products are 128 wide: a product of two shared-memory operands reads
// 4 KB of A per 16 channels whatever its width, which bounds 64 wide ones.
//
// Measured, bf16, 8192 rows, 16 heads, not causal: rows 765 us, columns 805 us
// at Dh = 128; 440 and 648 us at 64; 425 and 599 us at 32. At 128 the tensor
// cores are busy half the time, at 64 the exponentials' unit; what remains is
// the chain of a tile's steps.

#include <cuda_runtime.h>

#include <atomic>
#include <type_traits>

#include "fst_grouped_tc.cuh"

namespace fst {
namespace grouped {
namespace {

constexpr int kBM = 128;  // rows a block owns
constexpr int threads_of(int W) { return W * 128 + 64; }
constexpr int resident_of(int W) { return W == 1 ? 2 : 1; }

// Rows that see at most kFew keys take dS in two 16-bit parts, and one more
// product: all rows of an event of so few, the first ones of a causal event.
// With two keys dS_1 = -dS_2, and its rounding goes into dq whole; over more keys
// the roundings average out (error of dq over that of rounding dq itself: rows 1
// to 3 of a causal event 1.5, with the second part 1.1; from some 30 keys on 1.4
// whatever their number). Only the first tile of a block holds such rows, and only
// its first 32 keys (columns: query rows) need the second part: it lies between
// the first parts of those and of the next 32, which move up by kFewGap columns.
constexpr int kFew = 32, kFewGap = 16;
__device__ __forceinline__ bool few_keys(const FstGroupedProblem& p, const RowTile& t) {
  return t.len <= kFew || (p.causal && t.i0 == 0);
}
template <typename T>
__device__ __forceinline__ void store_rest(uint32_t dst, const float (&x)[32],
                                           const uint32_t (&rounded)[16]) {
  uint32_t w[16];
#pragma unroll
  for (int e = 0; e < 16; ++e)
    w[e] = Elem<T>::pack(x[2 * e] - Elem<T>::lo(rounded[e]), x[2 * e + 1] - Elem<T>::hi(rounded[e]));
  tmem_st16(dst, w);
}

// ---- the range of fp16 ------------------------------------------------------

template <typename T>
constexpr bool scaled() {
  return std::is_same<T, __half>::value;
}
constexpr int kPBits = 14;  // P <= 1 of the column kernel times 2^14

// Magnitudes of two fp16 values; 0 for those that are not finite, which make
// their own rows so whatever the powers, and must not shift those of others.
__device__ __forceinline__ uint32_t magnitudes(uint32_t w) {
  w &= 0x7fff7fff;
  return w & __vcmpltu2(w, 0x7c007c00);
}
// Largest finite |dO| and |v| of a block's 128 rows of an event and key head (all
// query heads of the group), as fp16 bits, low and high half of the word at the
// block's first row in ranges[kv_heads][rows].
__global__ void __launch_bounds__(256) range_kernel(const FstGroupedBackwardArgs a, int blocks,
                                                    uint32_t* ranges) {
  const FstGroupedProblem& p = a.prob;
  const int kh = blockIdx.x / blocks, group = p.heads / p.kv_heads;
  RowTile t;
  if (!find_tile<kBM>(p, blockIdx.x - kh * blocks, false, t) || t.i0 >= t.len) return;
  const int vecs = p.head_dim / 8, n = min(kBM, t.len - t.i0) * vecs;
  auto largest = [&](const FstRows& x, int h, uint32_t m) {
    for (int e = threadIdx.x; e < n; e += 256) {
      const uint4 w = *(const uint4*)(row_ptr<__half>(x, t, h, t.i0 + e / vecs) + e % vecs * 8);
      m = __vmaxu2(__vmaxu2(m, __vmaxu2(magnitudes(w.x), magnitudes(w.y))),
                   __vmaxu2(magnitudes(w.z), magnitudes(w.w)));
    }
    return m;
  };
  uint32_t g = 0;
  const uint32_t v = largest(a.v, kh, 0);
  for (int h = kh * group; h < (kh + 1) * group; ++h) g = largest(a.dout, h, g);
  __shared__ uint32_t warps[8];
  const uint32_t gm = __reduce_max_sync(0xffffffffu, max(g & 0xffff, g >> 16));
  const uint32_t vm = __reduce_max_sync(0xffffffffu, max(v & 0xffff, v >> 16));
  if (threadIdx.x % 32 == 0) warps[threadIdx.x / 32] = gm | vm << 16;
  __syncthreads();
  if (threadIdx.x == 0) {
    uint32_t m = 0;
    for (int i = 0; i < 8; ++i) m = __vmaxu2(m, warps[i]);
    ranges[stat_at(p, t, p.kv_heads, kh, t.i0)] = m;
  }
}
// The same of the whole event (whole warps).
__device__ __forceinline__ uint32_t event_range(const uint32_t* ranges, const FstGroupedProblem& p,
                                                const RowTile& t, int kh, int lane) {
  const uint32_t* at = ranges + stat_at(p, t, p.kv_heads, kh, 0);
  uint32_t m = 0;
  for (int64_t i = lane * kBM; i < t.len; i += 32 * kBM) m = __vmaxu2(m, at[i]);
  return __reduce_max_sync(0xffffffffu, m & 0xffff) |
         __reduce_max_sync(0xffffffffu, m >> 16) << 16;
}
__device__ __forceinline__ float half_bits(uint32_t x) {
  return __half2float(__ushort_as_half((unsigned short)x));
}
// Largest a for which 2^a 2 D g v stays below 2^15 (-26 to 61).
__device__ __forceinline__ int power_of(int D, float g, float v) {
  const float bound = fmaxf(2.f * D * g * v, 0x1p-47f);  // at most 2^40
  return 15 + 126 - (__float_as_int(bound) >> 23);  // bound < 2^((bits >> 23) - 126)
}
__device__ __forceinline__ float exp2i(int a) { return __int_as_float((a + 127) << 23); }

// ---- dq ---------------------------------------------------------------------

// The sum of dS over a row's keys is 0 before the rounding to 16 bits (and but
// for that of D) and not after, and an offset that all keys share would reach dq
// times that: keys of mean 2 (8) and deviation 1 left dq of 256 keys off by 3 (11)
// times one rounding of it, keys of mean 0 by 1.45. So a row c is taken off all
// keys, which changes nothing but that: the mean of the event's first 16, rounded
// to the type (then 1.45 for all three).
// A product of dS with ones sums the rows up, and the sum times c is taken off when
// the result is stored (dq of 256 short events 261 -> 285 us, 16384 causal of 64
// 522 -> 530, documents of 128 187 -> 192, 8192 rows of 16 heads 738 -> 765). c in
// registers by the time the products end: read from shared memory then, 302 for the
// short events. A product of dS with rows of -c in place of the sums: 281, and 534 for
// the long one, whose pass at the power limit takes 2 % more.
template <int Boxes, int W, int Stages>
struct RowSmem {
  alignas(1024) char q[Boxes * kBM * 128];
  alignas(1024) char g[Boxes * kBM * 128];
  alignas(1024) char k[Stages][Boxes * W * 64 * 128];
  alignas(1024) char v[Stages][Boxes * W * 64 * 128];
  // At two groups 1 KB more than this would take the next larger share of L1 (dq of
  // documents 187 -> 201 us).
  float delta[2][kBM];  // the groups' shares of D
  union {               // the first until all have read it
    uint16_t peak[2][kBM];  // and of max|dO| (fp16)
    Ones ones;
  };
  alignas(16) uint32_t c[Boxes * 32];
  uint64_t own_full, full[Stages], empty[Stages], s_full, s_free, dp_full, ds_ready, c_full, done;
  uint32_t tmem;
};

template <typename T, int Boxes, int W, int Stages>
__global__ void __launch_bounds__(threads_of(W), resident_of(W))
    dq_kernel(const __grid_constant__ TileMaps maps, const FstGroupedBackwardArgs a, int blocks,
              float* stats, const uint32_t* ranges) {
  using Smem = RowSmem<Boxes, W, Stages>;
  extern __shared__ char raw[];
  Smem& sm = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  constexpr int kBN = W * 64, kCols = W * 256, kTma = W * 4, kMma = kTma + 1;
  static_assert(W == 1 || sizeof(Smem) + 2048 <= 196 * 1024, "leaves L1 its share (RowSmem)");
  const FstGroupedProblem& p = a.prob;
  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (warp == kTma && lane == 0) {
    mbar_init(smem_addr(&sm.own_full), 1);
    for (int s = 0; s < Stages; ++s) {
      mbar_init(smem_addr(&sm.full[s]), 1);
      mbar_init(smem_addr(&sm.empty[s]), 1);
    }
    mbar_init(smem_addr(&sm.s_full), 1);
    mbar_init(smem_addr(&sm.s_free), W * 4);
    mbar_init(smem_addr(&sm.dp_full), 1);
    mbar_init(smem_addr(&sm.ds_ready), W * 4);
    mbar_init(smem_addr(&sm.c_full), 1);
    mbar_init(smem_addr(&sm.done), 1);
    mbar_init_fence();
    prefetch_map(&maps.q);
    prefetch_map(&maps.g);
    prefetch_map(&maps.k);
    prefetch_map(&maps.v);
  }
  __syncwarp();
  const BlockAt at = block_at(p, blocks, blockIdx.x);
  RowTile t;
  if (!find_tile<kBM>(p, at.id, p.causal, t)) return;
  const int D = p.head_dim;
  zero_dead_rows<T, kBM>(a.dq, t, at.h, D, threads_of(W));
  if (t.i0 >= t.len) return;
  const int end = p.causal ? min(t.len, t.i0 + kBM) : t.len;
  const int tiles = (end + kBN - 1) / kBN;

  auto load = [&](int it) {
    const int s = it % Stages;
    const uint32_t full = smem_addr(&sm.full[s]);
    mbar_arrive_tx(full, 2 * Boxes * kBN * 128);
    load_boxes<Boxes, kBN>(smem_addr(sm.k[s]), &maps.k, full, t.base + it * kBN, at.kh, t.ev);
    load_boxes<Boxes, kBN>(smem_addr(sm.v[s]), &maps.v, full, t.base + it * kBN, at.kh, t.ev);
  };
  if (warp == kTma && lane == 0) {
    // The first tiles set out before the others are ready for them.
    const uint32_t own = smem_addr(&sm.own_full);
    mbar_arrive_tx(own, 2 * Boxes * kBM * 128);
    load_boxes<Boxes, kBM>(smem_addr(sm.q), &maps.q, own, t.base + t.i0, at.h, t.ev);
    load_boxes<Boxes, kBM>(smem_addr(sm.g), &maps.g, own, t.base + t.i0, at.h, t.ev);
    for (int it = 0; it < Stages && it < tiles; ++it) load(it);
  }
  if (warp == kMma) tmem_alloc<kCols>(smem_addr(&sm.tmem));
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem;  // S, dP (dS over it), dQ, sums of dS

  bool ok = true;
  if (warp == kTma) {
    // Meanwhile c, two channels of each box a lane. (From the first tile: this
    // warp alone brings the next one into its place.)
    const int rows = min(t.len, 16);
    const float each = __fdividef(1.f, (float)rows);
    ok = mbar_wait(smem_addr(&sm.full[0]), 0);
#pragma unroll
    for (int b = 0; b < Boxes; ++b) {
      float x = 0.f, y = 0.f;
#pragma unroll 8
      for (int j = 0; j < rows; ++j) {
        const uint32_t w = *(const uint32_t*)(sm.k[0] + b * kBN * 128 + j * 128 +
                                              ((lane / 4) ^ (j & 7)) * 16 + lane % 4 * 4);
        x += Elem<T>::lo(w);
        y += Elem<T>::hi(w);
      }
      sm.c[b * 32 + lane] = Elem<T>::pack(x * each, y * each);
    }
    __syncwarp();
    if (lane == 0) {
      mbar_arrive(smem_addr(&sm.c_full));
      for (int it = Stages; it < tiles && ok; ++it) {
        ok = mbar_wait(smem_addr(&sm.empty[it % Stages]), (it / Stages - 1) & 1);
        if (ok) load(it);
      }
    }
  } else if (warp == kMma) {
    const uint32_t leader = elect_one();
    const int n = uniform(tiles), last = uniform(end), dim = uniform(D);
    const uint32_t s_mem = uniform(tmem), p_mem = s_mem + kBN, q_mem = p_mem + kBN,
                   sum_mem = q_mem + Boxes * 64;
    const uint32_t acc_instr = instruction<T>((dim + 15) & ~15, true, false);
    const bool few = uniform(few_keys(p, t));
    auto keys = [&](int it) { return min(kBN, last - it * kBN); };
    auto logits = [&](int it) {
      if (!mbar_wait(smem_addr(&sm.full[it % Stages]), (it / Stages) & 1)) return false;
      product<T, Boxes, kBM, kBN>(s_mem, smem_addr(sm.q), smem_addr(sm.k[it % Stages]), dim,
                                  (keys(it) + 15) & ~15, p.scale < 0.f, leader);
      tc_commit(smem_addr(&sm.s_full), leader);
      return true;
    };
    // Over dS: MMAs complete in order, so the product that read it is done.
    auto weights = [&](int it) {
      product<T, Boxes, kBM, kBN>(p_mem, smem_addr(sm.g), smem_addr(sm.v[it % Stages]), dim,
                                  (keys(it) + 15) & ~15, false, leader);
      tc_commit(smem_addr(&sm.dp_full), leader);
    };
    // The ones, while the first tiles are on their way, or when the groups have read
    // what lies there.
    constexpr bool kLate = W == 2 && scaled<T>();
    if (!kLate) {
      fill_ones<T>(sm.ones, lane);
      __syncwarp();
    }
    ok = mbar_wait(smem_addr(&sm.own_full), 0) && logits(0);
    if (ok) weights(0);
    for (int it = 0; it < n && ok; ++it) {
      if (it + 1 < n) {
        ok = mbar_wait(smem_addr(&sm.s_free), it & 1);
        tc_fence_after();
        ok = ok && logits(it + 1);
      }
      ok = ok && mbar_wait(smem_addr(&sm.ds_ready), it & 1);
      if (!ok) break;
      tc_fence_after();
      if (kLate && it == 0) {
        fill_ones<T>(sm.ones, lane);
        __syncwarp();
      }
      const bool second = few && it == 0;
      accumulate<kBN>(q_mem, p_mem, smem_addr(sm.k[it % Stages]), keys(it), acc_instr, it > 0,
                      leader, second ? kFewGap : 0);
      row_sums<T, kBN>(sum_mem, p_mem, smem_addr(&sm.ones), keys(it), it > 0, leader,
                       second ? kFewGap : 0);
      if (second) {
        accumulate<kBN>(q_mem, p_mem + kFewGap, smem_addr(sm.k[0]), min(last, kFew), acc_instr,
                        true, leader);
        row_sums<T, kBN>(sum_mem, p_mem + kFewGap, smem_addr(&sm.ones), min(last, kFew), true,
                         leader);
      }
      tc_commit(smem_addr(&sm.empty[it % Stages]), leader);
      if (it + 1 < n) weights(it + 1);
    }
    if (ok) tc_commit(smem_addr(&sm.done), leader);
  } else {
    const int w = warp / 4, row = warp % 4 * 32 + lane;  // key columns [64 w, +64) of a tile
    const uint32_t quad = (uint32_t)(warp % 4 * 32) << 16;
    const uint32_t tS = tmem + quad + w * 64, tP = tS + kBN;
    const int i = t.i0 + row;
    const bool live = i < t.len;
    const float c2 = fabsf(p.scale) * kLog2e;
    float lse2 = 0.f, delta = 0.f;
    uint32_t range = 0, peak = 0;
    if (scaled<T>()) range = event_range(ranges, p, t, at.kh, lane);
    if (live) {
      // Each group sums its 64 channels.
      const int d0 = w * 64, n = W == 1 ? D : min(D - d0, 64);
      const T* g = row_ptr<T>(a.dout, t, at.h, i) + d0;
      const T* o = row_ptr<T>(a.out, t, at.h, i) + d0;
      const T* r = a.out_low.data ? row_ptr<T>(a.out_low, t, at.h, i) + d0 : nullptr;
#pragma unroll 4
      for (int d = 0; d < n; d += 8) {
        const uint4 y = *(const uint4*)(g + d), x = *(const uint4*)(o + d);
        const uint4 z = r ? *(const uint4*)(r + d) : make_uint4(0, 0, 0, 0);
        const uint32_t ys[4] = {y.x, y.y, y.z, y.w}, xs[4] = {x.x, x.y, x.z, x.w},
                       zs[4] = {z.x, z.y, z.z, z.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          delta = fmaf(Elem<T>::lo(xs[e]) + Elem<T>::lo(zs[e]), Elem<T>::lo(ys[e]), delta);
          delta = fmaf(Elem<T>::hi(xs[e]) + Elem<T>::hi(zs[e]), Elem<T>::hi(ys[e]), delta);
          if (scaled<T>()) peak = __vmaxu2(peak, magnitudes(ys[e]));
        }
      }
    }
    if (W == 2) {
      sm.delta[w][row] = delta;
      if (scaled<T>()) sm.peak[w][row] = (uint16_t)max(peak & 0xffff, peak >> 16);
      tc::named_sync(1, W * 128);
      delta = sm.delta[0][row] + sm.delta[1][row];
      if (scaled<T>()) peak = max(sm.peak[0][row], sm.peak[1][row]);
    }
    if (live) {
      const int64_t st = stat_at(p, t, p.heads, at.h, i);
      lse2 = a.lse[st] * kLog2e;
      if (w == 0) {  // for the column kernel, in the form it adds them
        float shared = 1.f;
        if (scaled<T>())
          shared = exp2i(power_of(D, half_bits(range & 0xffff), half_bits(range >> 16)) - kPBits);
        stats[st] = scaled<T>() ? kPBits - lse2 : -lse2;
        stats[st + p.total_rows * p.heads] = -delta * shared;
      }
    }
    float undo = p.scale;
    if (scaled<T>()) {
      const int power = power_of(D, half_bits(max(peak & 0xffff, peak >> 16)),
                                 half_bits(range >> 16));
      lse2 -= power;
      undo *= exp2i(-power);
    }
    const pair_t scale2 = pair(c2, c2), lse2n = pair(-lse2, -lse2), delta2n = pair(-delta, -delta);
    // One tile. `Whole`: every row of the block sees all its keys.
    auto tile = [&](auto whole, auto is_few, int it) {
      constexpr bool Whole = decltype(whole)::value, Few = decltype(is_few)::value;
      const int j0 = it * kBN + w * 64, nk = end - j0;
      if (!mbar_wait(smem_addr(&sm.s_full), it & 1)) return false;
      tc_fence_after();
      float s[2][32];
      if (Whole || nk > 0) tmem_ld32(s[0], tS);
      if (Whole || nk > 32) tmem_ld32(s[1], tS + 32);
      tmem_wait_ld();
      pin(s[0]);
      pin(s[1]);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_addr(&sm.s_free));
#pragma unroll
      for (int e = 0; e < 64; e += 2) {
        float* x = &s[e / 32][e % 32];
        const float2 y = split(fma2(pair(x[0], x[1]), scale2, lse2n));
        x[0] = ex2(y.x);
        x[1] = ex2(y.y);
      }
      if (!mbar_wait(smem_addr(&sm.dp_full), it & 1)) return false;
      tc_fence_after();
      // Keys below lim are seen; the warp's first row sees fewest. A row that
      // sees one key has P = 1 and dP = D, so its dS is 0: formed from two
      // sums of different order it would be their rounding.
      const int keys = p.causal ? min(i + 1, t.len) : t.len;
      const int lim = (keys > 1 ? keys : 0) - j0;
      const int fewest = Whole ? 64 : uniform(lim);
      const bool second = Few && w == 0;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        if (!Whole && c * 32 >= nk) continue;
        float dp[32];
        tmem_ld32(dp, tP + c * 32);
        tmem_wait_ld();
        pin(dp);
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const float2 x = split(
              mul2(pair(s[c][e], s[c][e + 1]), add2(pair(dp[e], dp[e + 1]), delta2n)));
          dp[e] = x.x;
          dp[e + 1] = x.y;
        }
        if (!Whole && c * 32 + 32 > fewest) {
#pragma unroll
          for (int e = 0; e < 32; ++e) dp[e] = c * 32 + e < lim ? dp[e] : 0.f;
        }
        uint32_t x[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = Elem<T>::pack(dp[2 * e], dp[2 * e + 1]);
        tmem_st16(tP + c * (second ? 16 + kFewGap : 16), x);
        if (second && c == 0) store_rest<T>(tP + kFewGap, dp, x);
      }
      const int all = min(kBN, end - it * kBN);
      if (!Whole && (all & 15))  // dS is 0 there, and must not meet another event's NaN
        zero_tile_rows<Boxes, kBN>(sm.k[it % Stages], all, (all + 15) & ~15, threadIdx.x, W * 128);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_addr(&sm.ds_ready));
      return true;
    };
    const int whole = min(tiles, (p.causal ? min(t.len, t.i0 + 1) : t.len) / kBN);
    int it = 0;
    for (; it < whole && ok; ++it) ok = tile(std::true_type(), std::false_type(), it);
    if (few_keys(p, t)) ok = tile(std::false_type(), std::true_type(), it++);
    for (; it < tiles && ok; ++it) ok = tile(std::false_type(), std::false_type(), it);
    uint32_t c[32];
    ok = ok && mbar_wait(smem_addr(&sm.c_full), 0);
#pragma unroll
    for (int e = 0; e < 32; e += 4) {
      const uint4 x = *(const uint4*)(sm.c + w * 32 + e);
      c[e] = x.x;
      c[e + 1] = x.y;
      c[e + 2] = x.z;
      c[e + 3] = x.w;
    }
    ok = ok && mbar_wait(smem_addr(&sm.done), 0);
    tc_fence_after();
    // The groups share the columns of the result.
    store_row_less<T>(live ? row_ptr<T>(a.dq, t, at.h, i) + w * 64 : nullptr,
                      tmem + quad + 2 * kBN + w * 64, W == 1 ? D : min(D - w * 64, 64),
                      ok ? undo : NAN, c, tmem + quad + 2 * kBN + Boxes * 64);
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  if (warp == kMma) tmem_free<kCols>(tmem);
}

// ---- dk, dv -----------------------------------------------------------------

template <int Boxes, int W, int Stages>
struct ColSmem {
  alignas(1024) char k[Boxes * kBM * 128];
  alignas(1024) char v[Boxes * kBM * 128];
  alignas(1024) char q[Stages][Boxes * W * 64 * 128];
  alignas(1024) char g[Stages][Boxes * W * 64 * 128];
  alignas(16) float lse2n[Stages][W * 64];   // -log2(e) lse of the query rows
  alignas(16) float deltan[Stages][W * 64];  // -D
  uint64_t own_full, full[Stages], empty[Stages], s_full, p_ready, dp_full, ds_ready, done;
  uint32_t tmem;
};

template <typename T, int Boxes, int W, int Stages>
__global__ void __launch_bounds__(threads_of(W), resident_of(W))
    dkv_kernel(const __grid_constant__ TileMaps maps, const FstGroupedBackwardArgs a, int blocks,
               const float* stats, const uint32_t* ranges) {
  using Smem = ColSmem<Boxes, W, Stages>;
  extern __shared__ char raw[];
  Smem& sm = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  constexpr int kBN = W * 64, kAcc = Boxes * 64;  // query rows a tile; columns of dV and of dK
  constexpr int kCols = 2 * kBN + 2 * kAcc;       // 256 or 512
  constexpr int kTma = W * 4, kMma = kTma + 1;    // warps
  static_assert(kCols == 256 || kCols == 512, "tensor memory comes in powers of two");
  const FstGroupedProblem& p = a.prob;
  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (warp == kTma && lane == 0) {
    mbar_init(smem_addr(&sm.own_full), 1);
    for (int s = 0; s < Stages; ++s) {
      mbar_init(smem_addr(&sm.full[s]), 1 + 32);  // TMA, and each lane's copies
      mbar_init(smem_addr(&sm.empty[s]), 1);
    }
    mbar_init(smem_addr(&sm.s_full), 1);
    mbar_init(smem_addr(&sm.p_ready), W * 4);
    mbar_init(smem_addr(&sm.dp_full), 1);
    mbar_init(smem_addr(&sm.ds_ready), W * 4);
    mbar_init(smem_addr(&sm.done), 1);
    mbar_init_fence();
    prefetch_map(&maps.q);
    prefetch_map(&maps.g);
    prefetch_map(&maps.k);
    prefetch_map(&maps.v);
  }
  __syncwarp();
  const int kh = blockIdx.x / blocks, id = blockIdx.x - kh * blocks;
  const int group = p.heads / p.kv_heads;
  RowTile t;
  if (!find_tile<kBM>(p, id, false, t)) return;
  const int D = p.head_dim;
  zero_dead_rows<T, kBM>(a.dk, t, kh, D, threads_of(W));
  zero_dead_rows<T, kBM>(a.dv, t, kh, D, threads_of(W));
  if (t.i0 >= t.len) return;
  const int first = p.causal ? t.i0 : 0;                 // first query row
  const int per_head = (t.len - first + kBN - 1) / kBN;  // query tiles a head
  const int tiles = per_head * group;

  if (warp == kTma && lane == 0) {
    const uint32_t own = smem_addr(&sm.own_full);
    mbar_arrive_tx(own, 2 * Boxes * kBM * 128);
    load_boxes<Boxes, kBM>(smem_addr(sm.k), &maps.k, own, t.base + t.i0, kh, t.ev);
    load_boxes<Boxes, kBM>(smem_addr(sm.v), &maps.v, own, t.base + t.i0, kh, t.ev);
  }
  if (warp == kMma) tmem_alloc<kCols>(smem_addr(&sm.tmem));
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem;  // S^T (P^T over it), dP^T (dS^T over it), dV, dK

  bool ok = true;
  if (warp == kTma) {
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
      const float* st = stats + stat_at(p, t, p.heads, h, q0);
#pragma unroll
      for (int r = lane; r < kBN; r += 32) {
        const bool live = q0 + r < t.len;
        const float* src = live ? st + r : stats;
        copy4(smem_addr(&sm.lse2n[s][r]), src, live);
        copy4(smem_addr(&sm.deltan[s][r]), src + (live ? p.total_rows * p.heads : 0), live);
      }
      async_arrive(full);
      q0 += kBN;
      if (q0 >= t.len) {
        q0 = first;
        ++h;
      }
    }
  } else if (warp == kMma) {
    const uint32_t leader = elect_one();
    const int n = uniform(tiles), rows = uniform(t.len - first), dim = uniform(D);
    const uint32_t s_mem = uniform(tmem), p_mem = s_mem + kBN, v_mem = p_mem + kBN,
                   k_mem = v_mem + kAcc;
    const uint32_t acc_instr = instruction<T>((dim + 15) & ~15, true, false);
    const bool few = uniform(few_keys(p, t));
    // S^T over P^T and dP^T over dS^T: MMAs complete in order, so the products
    // that read those are done.
    auto logits = [&](int it, int q_rows) {
      if (!mbar_wait(smem_addr(&sm.full[it % Stages]), (it / Stages) & 1)) return false;
      product<T, Boxes, kBM, kBN>(s_mem, smem_addr(sm.k), smem_addr(sm.q[it % Stages]), dim,
                                  (q_rows + 15) & ~15, p.scale < 0.f, leader);
      tc_commit(smem_addr(&sm.s_full), leader);
      return true;
    };
    auto weights = [&](int it, int q_rows) {
      product<T, Boxes, kBM, kBN>(p_mem, smem_addr(sm.v), smem_addr(sm.g[it % Stages]), dim,
                                  (q_rows + 15) & ~15, false, leader);
      tc_commit(smem_addr(&sm.dp_full), leader);
    };
    int done = 0, q_rows = min(kBN, rows);  // query rows of the head behind, of the tile
    ok = mbar_wait(smem_addr(&sm.own_full), 0) && logits(0, q_rows);
    if (ok) weights(0, q_rows);
    for (int it = 0; it < n && ok; ++it) {
      const int s = it % Stages;
      const bool second = few && done == 0;  // a head's first tile
      done = done + kBN < rows ? done + kBN : 0;
      const int next_rows = min(kBN, rows - done);
      ok = mbar_wait(smem_addr(&sm.p_ready), it & 1);
      if (!ok) break;
      tc_fence_after();
      accumulate<kBN>(v_mem, s_mem, smem_addr(sm.g[s]), q_rows, acc_instr, it > 0, leader);
      if (it + 1 < n) ok = logits(it + 1, next_rows);
      ok = ok && mbar_wait(smem_addr(&sm.ds_ready), it & 1);
      if (!ok) break;
      tc_fence_after();
      accumulate<kBN>(k_mem, p_mem, smem_addr(sm.q[s]), q_rows, acc_instr, it > 0, leader,
                      second ? kFewGap : 0);
      if (second)
        accumulate<kBN>(k_mem, p_mem + kFewGap, smem_addr(sm.q[s]), min(q_rows, kFew), acc_instr,
                        true, leader);
      tc_commit(smem_addr(&sm.empty[s]), leader);
      if (it + 1 < n) weights(it + 1, next_rows);
      q_rows = next_rows;
    }
    if (ok) tc_commit(smem_addr(&sm.done), leader);
  } else {
    const int w = warp / 4;  // query columns [64 w, +64) of a tile
    const uint32_t quad = (uint32_t)(warp % 4 * 32) << 16;
    const uint32_t tS = tmem + quad + w * 64, tP = tS + kBN;
    const int j = t.i0 + warp % 4 * 32 + lane;
    const float c2 = fabsf(p.scale) * kLog2e;
    const pair_t scale2 = pair(c2, c2);
    // dS 2^power from P 2^kPBits: the factor left for dP (and, by the row
    // kernel, for D).
    int power = 0;
    if (scaled<T>()) {
      const uint32_t range = event_range(ranges, p, t, kh, lane);
      power = power_of(D, half_bits(range & 0xffff), half_bits(range >> 16));
    }
    const float rest = exp2i(power - kPBits);
    const pair_t rest2 = pair(rest, rest);
    for (int it = 0, q0 = first; it < tiles; ++it, q0 = q0 + kBN < t.len ? q0 + kBN : first) {
      const int s = it % Stages, all = min(kBN, t.len - q0);
      const int qw = q0 + w * 64, nq = t.len - qw;  // this group's columns
      const bool edge = nq < 64 || (p.causal && qw < t.i0 + kBM - 1);
      const int lo = p.causal ? j - qw : 0;  // columns lo <= c < nq see key j
      // Row 0 of a causal event, and the row of an event of one, see one key:
      // dS is 0 (see the row kernel).
      const int ds_lo = p.causal ? max(lo, 1 - qw) : t.len > 1 ? 0 : 1;
      const float* ls = &sm.lse2n[s][w * 64];
      const float* de = &sm.deltan[s][w * 64];
      ok = mbar_wait(smem_addr(&sm.full[s]), (it / Stages) & 1);
      ulonglong2 ahead[8];  // the first half's statistics, read before they are needed
#pragma unroll
      for (int e = 0; e < 8; ++e) ahead[e] = *(const ulonglong2*)(ls + e * 4);
      ok = ok && mbar_wait(smem_addr(&sm.s_full), it & 1);
      if (!ok) break;
      tc_fence_after();
      float x[2][32];
#pragma unroll
      for (int c = 0; c < 2; ++c)
        if (c * 32 < nq) tmem_ld32(x[c], tS + c * 32);
      tmem_wait_ld();
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        if (c * 32 >= nq) continue;
        pin(x[c]);
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          const ulonglong2 l4 = c ? *(const ulonglong2*)(ls + c * 32 + e) : ahead[e / 4];
#pragma unroll
          for (int f = 0; f < 4; f += 2) {
            const float2 y =
                split(fma2(pair(x[c][e + f], x[c][e + f + 1]), scale2, f ? l4.y : l4.x));
            x[c][e + f] = ex2(y.x);
            x[c][e + f + 1] = ex2(y.y);
          }
        }
        if (edge) {
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const int col = c * 32 + e;
            x[c][e] = col >= lo && col < nq ? x[c][e] : 0.f;
          }
        }
        uint32_t y[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) y[e] = Elem<T>::pack(x[c][2 * e], x[c][2 * e + 1]);
        tmem_st16(tS + c * 16, y);
      }
      if (all & 15) {
        // Rows up to the next multiple of 16 have P = dS = 0, and must not meet
        // another event's NaN. dP^T has to have read dO by then.
        ok = mbar_wait(smem_addr(&sm.dp_full), it & 1);
        if (!ok) break;
        zero_tile_rows<Boxes, kBN>(sm.q[s], all, (all + 15) & ~15, threadIdx.x, W * 128);
        zero_tile_rows<Boxes, kBN>(sm.g[s], all, (all + 15) & ~15, threadIdx.x, W * 128);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_addr(&sm.p_ready));
#pragma unroll
      for (int e = 0; e < 8; ++e) ahead[e] = *(const ulonglong2*)(de + e * 4);
      ok = mbar_wait(smem_addr(&sm.dp_full), it & 1);
      if (!ok) break;
      tc_fence_after();
      const bool second = w == 0 && q0 == first && few_keys(p, t);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        if (c * 32 >= nq) continue;
        float dp[32];
        tmem_ld32(dp, tP + c * 32);
        tmem_wait_ld();
        pin(dp);
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          const ulonglong2 d4 = c ? *(const ulonglong2*)(de + c * 32 + e) : ahead[e / 4];
#pragma unroll
          for (int f = 0; f < 4; f += 2) {
            const pair_t p2 = pair(dp[e + f], dp[e + f + 1]), d2 = f ? d4.y : d4.x;
            const float2 y = split(mul2(pair(x[c][e + f], x[c][e + f + 1]),
                                        scaled<T>() ? fma2(p2, rest2, d2) : add2(p2, d2)));
            dp[e + f] = y.x;
            dp[e + f + 1] = y.y;
          }
        }
        if (edge) {
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const int col = c * 32 + e;
            dp[e] = col >= ds_lo && col < nq ? dp[e] : 0.f;
          }
        }
        uint32_t y[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) y[e] = Elem<T>::pack(dp[2 * e], dp[2 * e + 1]);
        tmem_st16(tP + c * (second ? 16 + kFewGap : 16), y);
        if (second && c == 0) store_rest<T>(tP + kFewGap, dp, y);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_addr(&sm.ds_ready));
    }
    if (ok) ok = mbar_wait(smem_addr(&sm.done), 0);
    tc_fence_after();
    // One of two groups stores dV, the other dK.
    const bool live = j < t.len;
    const uint32_t tV = tmem + quad + 2 * kBN, tK = tV + kAcc;
    if (w == 0)
      store_row<T>(live ? row_ptr<T>(a.dv, t, kh, j) : nullptr, tV, D,
                   ok ? exp2i(scaled<T>() ? -kPBits : 0) : NAN);
    if (w == W - 1)
      store_row<T>(live ? row_ptr<T>(a.dk, t, kh, j) : nullptr, tK, D,
                   ok ? p.scale * exp2i(-power) : NAN);
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  if (warp == kMma) tmem_free<kCols>(tmem);
}

template <typename K>
int prepare(K kernel, int bytes, std::atomic<uint64_t>& done) {
  const int e = allow_dynamic_smem((const void*)kernel, bytes, done);
  if (e) return api_fail(FST_ERR_CUDA, "shared memory: %s", cudaGetErrorString((cudaError_t)e));
  return FST_OK;
}

template <typename T, int Boxes, int W, int RowStages, int ColStages>
int launch(const FstGroupedBackwardArgs& a, cudaStream_t st) {
  const FstGroupedProblem& p = a.prob;
  static std::atomic<uint64_t> row_done{0}, col_done{0};
  const auto rows_k = dq_kernel<T, Boxes, W, RowStages>;
  const auto cols_k = dkv_kernel<T, Boxes, W, ColStages>;
  const int row_bytes = (int)sizeof(RowSmem<Boxes, W, RowStages>) + 1024;
  const int col_bytes = (int)sizeof(ColSmem<Boxes, W, ColStages>) + 1024;
  int rc = prepare(rows_k, row_bytes, row_done);
  if (!rc) rc = prepare(cols_k, col_bytes, col_done);
  const int64_t rows = p.packed ? p.total_rows : p.max_len, events = p.packed ? 1 : p.batch;
  const int D = p.head_dim, other = W * 64;
  TileMaps r, c;  // 128 own rows, 64 W of the other side
  if (!rc) rc = tc::make_rows_map(&r.q, a.q, D, rows, p.heads, events, kBM);
  if (!rc) rc = tc::make_rows_map(&r.g, a.dout, D, rows, p.heads, events, kBM);
  if (!rc) rc = tc::make_rows_map(&r.k, a.k, D, rows, p.kv_heads, events, other);
  if (!rc) rc = tc::make_rows_map(&r.v, a.v, D, rows, p.kv_heads, events, other);
  if (!rc && W == 2) c = r;  // the same boxes
  if (!rc && W == 1) rc = tc::make_rows_map(&c.q, a.q, D, rows, p.heads, events, other);
  if (!rc && W == 1) rc = tc::make_rows_map(&c.g, a.dout, D, rows, p.heads, events, other);
  if (!rc && W == 1) rc = tc::make_rows_map(&c.k, a.k, D, rows, p.kv_heads, events, kBM);
  if (!rc && W == 1) rc = tc::make_rows_map(&c.v, a.v, D, rows, p.kv_heads, events, kBM);
  if (rc) return rc;
  const int blocks = (int)list_blocks(p, kBM);
  uint32_t* ranges = reinterpret_cast<uint32_t*>(a.stats + 2 * p.total_rows * p.heads);
  if (scaled<T>()) {
    range_kernel<<<(unsigned)(blocks * p.kv_heads), 256, 0, st>>>(a, blocks, ranges);
    count_launch();
  }
  rows_k<<<(unsigned)(blocks * p.heads), threads_of(W), row_bytes, st>>>(r, a, blocks, a.stats,
                                                                         ranges);
  cols_k<<<(unsigned)(blocks * p.kv_heads), threads_of(W), col_bytes, st>>>(c, a, blocks, a.stats,
                                                                            ranges);
  count_launch(2);
  return FST_OK;
}

template <typename T>
int launch_t(const FstGroupedBackwardArgs& a, cudaStream_t st) {
  if (a.prob.head_dim <= 64) return launch<T, 1, 1, 3, 4>(a, st);
  return launch<T, 2, 2, 2, 2>(a, st);
}

}  // namespace

bool tc_takes(const FstGroupedBackwardArgs& a) {
  const FstGroupedProblem& p = a.prob;
  return tc_type(p) && on_grid(p, a.q, p.heads) && on_grid(p, a.out, p.heads) &&
         (!a.out_low.data || on_grid(p, a.out_low, p.heads)) && on_grid(p, a.dout, p.heads) && on_grid(p, a.dq, p.heads) &&
         on_grid(p, a.k, p.kv_heads) && on_grid(p, a.v, p.kv_heads) &&
         on_grid(p, a.dk, p.kv_heads) && on_grid(p, a.dv, p.kv_heads);
}

int tc_backward(const FstGroupedBackwardArgs& a, cudaStream_t st) {
  if (a.prob.dtype == FST_BF16) return launch_t<__nv_bfloat16>(a, st);
  return launch_t<__half>(a, st);
}

}  // namespace grouped
}  // namespace fst
