// Grouped-head attention on the 5th-generation tensor cores: the pieces that
// its forward and backward kernels share (tcgen05, TMEM, TMA, work order).
//
// A tile is rows of one head's [rows, Dh] slice, brought by TMA in boxes of 64
// channels (128 bytes a row, 128-byte swizzle); channels past Dh and rows past
// the tensor read as zeros, so every Dh that is a multiple of 8 up to 128
// runs on the same code, with one box (Dh <= 64) or two. Products use
// kind::f16 with fp32 accumulators in tensor memory.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "fst_grouped.cuh"
#include "fst_tc_common.cuh"

namespace fst {
namespace grouped {

using tc::Elem;
using tc::ex2;
using tc::fence_proxy_async;
using tc::mbar_arrive_tx;
using tc::mbar_init;
using tc::mbar_init_fence;
using tc::mbar_wait;

// Tensor maps of a launch (make_rows_map), passed as a kernel parameter.
struct __align__(64) TileMaps {
  CUtensorMap q, k, v, g;
};

// ---- tcgen05 ----------------------------------------------------------------

__device__ __forceinline__ uint32_t smem_addr(const void* p) {
  return (uint32_t)__cvta_generic_to_shared(p);
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Whole warp. The address of the allocation is written to `slot`.
template <int Cols>
__device__ __forceinline__ void tmem_alloc(uint32_t slot) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot),
               "n"(Cols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
template <int Cols>
__device__ __forceinline__ void tmem_free(uint32_t addr) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "n"(Cols));
}
__device__ __forceinline__ void tc_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
// One lane of a converged warp.
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t leader;
  asm volatile(
      "{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}"
      : "=r"(leader));
  return leader;
}
// A value that is the same in every lane, in a form the compiler knows to be.
// The issuing warp runs converged, on such values, and leaves the choice of
// the issuing lane to a predicate on each instruction: descriptors are then
// formed on the uniform datapath (a lane's branch of its own costs about 100
// cycles an MMA to move them there).
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }

// Arrives on `bar` when every MMA the leader has issued so far is complete.
__device__ __forceinline__ void tc_commit(uint32_t bar, uint32_t leader) {
  asm volatile(
      "{\n .reg .pred e;\n setp.ne.b32 e, %1, 0;\n"
      " @e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}" ::"r"(
          bar),
      "r"(leader)
      : "memory");
}

// Shared-memory operand in the 128-byte swizzle: start address, leading and
// stride byte offsets in units of 16 bytes, descriptor version 1.
// K-major (rows of 64 channels, the product runs along the channels): 8-row
// groups are 1024 bytes apart. MN-major (the product runs along the rows): the
// same 8-row groups are the stride, and `lead` separates boxes of 64 channels.
__device__ __forceinline__ uint64_t operand(uint32_t addr, uint32_t lead) {
  return (uint64_t)((addr >> 4) & 0x3fff) | (uint64_t)((lead >> 4) & 0x3fff) << 16 |
         (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// Instruction descriptor: fp32 accumulator, A and B of type T, M = 128.
template <typename T>
__device__ __forceinline__ uint32_t instruction(int n, bool b_mn_major, bool negate) {
  const uint32_t type = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
  return 1u << 4 | type << 7 | type << 10 | (negate ? 1u << 13 : 0) |
         (b_mn_major ? 1u << 16 : 0) | (uint32_t)(n >> 3) << 17 | (128u >> 4) << 24;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                       bool add, uint32_t leader) {
  asm volatile(
      "{\n .reg .pred p, e;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 e, %5, 0;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((int)add), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                       bool add, uint32_t leader) {
  asm volatile(
      "{\n .reg .pred p, e;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 e, %5, 0;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"((int)add), "r"(leader)
      : "memory");
}

// 32 columns of the warp's 32 lanes (one row a thread). The values may be
// read after tmem_wait_ld().
__device__ __forceinline__ void tmem_ld32(float (&r)[32], uint32_t addr) {
  uint32_t* x = reinterpret_cast<uint32_t*>(r);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]), "=r"(x[4]), "=r"(x[5]), "=r"(x[6]),
        "=r"(x[7]), "=r"(x[8]), "=r"(x[9]), "=r"(x[10]), "=r"(x[11]), "=r"(x[12]), "=r"(x[13]),
        "=r"(x[14]), "=r"(x[15]), "=r"(x[16]), "=r"(x[17]), "=r"(x[18]), "=r"(x[19]),
        "=r"(x[20]), "=r"(x[21]), "=r"(x[22]), "=r"(x[23]), "=r"(x[24]), "=r"(x[25]),
        "=r"(x[26]), "=r"(x[27]), "=r"(x[28]), "=r"(x[29]), "=r"(x[30]), "=r"(x[31])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&x)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr),
      "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(x[4]), "r"(x[5]), "r"(x[6]), "r"(x[7]),
      "r"(x[8]), "r"(x[9]), "r"(x[10]), "r"(x[11]), "r"(x[12]), "r"(x[13]), "r"(x[14]),
      "r"(x[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
// One column; may be used after tmem_wait_ld(), and a pin.
__device__ __forceinline__ float tmem_ld1(uint32_t addr) {
  float x;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=f"(x) : "r"(addr) : "memory");
  return x;
}
__device__ __forceinline__ void pin(float& x) { asm volatile("" : "+f"(x)); }
// 16 columns in place: each row times its factor. Waits for itself.
__device__ __forceinline__ void tmem_scale16(uint32_t addr, float f) {
  uint32_t x[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]), "=r"(x[4]), "=r"(x[5]), "=r"(x[6]),
        "=r"(x[7]), "=r"(x[8]), "=r"(x[9]), "=r"(x[10]), "=r"(x[11]), "=r"(x[12]), "=r"(x[13]),
        "=r"(x[14]), "=r"(x[15])
      : "r"(addr)
      : "memory");
#pragma unroll
  for (int e = 0; e < 16; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) * f);
  tmem_st16(addr, x);
}
// Keeps the uses of loaded registers behind the tmem_wait_ld() before it.
__device__ __forceinline__ void pin(float (&x)[32]) {
  asm volatile(""
               : "+f"(x[0]), "+f"(x[1]), "+f"(x[2]), "+f"(x[3]), "+f"(x[4]), "+f"(x[5]),
                 "+f"(x[6]), "+f"(x[7]), "+f"(x[8]), "+f"(x[9]), "+f"(x[10]), "+f"(x[11]),
                 "+f"(x[12]), "+f"(x[13]), "+f"(x[14]), "+f"(x[15]));
  asm volatile(""
               : "+f"(x[16]), "+f"(x[17]), "+f"(x[18]), "+f"(x[19]), "+f"(x[20]), "+f"(x[21]),
                 "+f"(x[22]), "+f"(x[23]), "+f"(x[24]), "+f"(x[25]), "+f"(x[26]), "+f"(x[27]),
                 "+f"(x[28]), "+f"(x[29]), "+f"(x[30]), "+f"(x[31]));
}
__device__ __forceinline__ void tmem_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// ---- pairs of fp32 values (one instruction for two lanes' worth) -------------

using pair_t = unsigned long long;
__device__ __forceinline__ pair_t pair(float a, float b) {
  pair_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 split(pair_t x) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
  return r;
}
__device__ __forceinline__ pair_t fma2(pair_t a, pair_t b, pair_t c) {
  pair_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ pair_t add2(pair_t a, pair_t b) {
  pair_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ pair_t mul2(pair_t a, pair_t b) {
  pair_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// A NaN among the three is the result.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// ---- TMA --------------------------------------------------------------------

__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}
// Box of 64 channels from `c` (a multiple of 64: 128 bytes), rows from `row`
// of head `h` of event `ev`. Rows and channels past the tensor read as zeros.
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c,
                                         int row, int h, int ev) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];\n" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c), "r"(row), "r"(h), "r"(ev)
      : "memory");
}
// All boxes of a tile of `Rows` rows; Boxes * Rows * 128 bytes land on `bar`.
template <int Boxes, int Rows>
__device__ __forceinline__ void load_boxes(uint32_t dst, const CUtensorMap* map, uint32_t bar,
                                           int row, int h, int ev) {
#pragma unroll
  for (int b = 0; b < Boxes; ++b) load_box(dst + b * Rows * 128, map, bar, b * 64, row, h, ev);
}

// Four bytes from global to shared memory, or zero; lands on the barrier that
// async_arrive names (one arrival of each thread).
__device__ __forceinline__ void copy4(uint32_t dst, const float* src, bool live) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src),
               "r"(live ? 4 : 0)
               : "memory");
}
__device__ __forceinline__ void async_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

// Zeros rows [first, last) of a tile (whole rows, so the swizzle does not
// matter), by `n` threads of index t; made visible to the tensor cores.
template <int Boxes, int Rows>
__device__ __forceinline__ void zero_tile_rows(char* tile, int first, int last, int t, int n) {
  for (int e = t; e < (last - first) * 8 * Boxes; e += n) {
    const int b = e / ((last - first) * 8), r = e - b * (last - first) * 8;
    *(uint4*)(tile + b * Rows * 128 + first * 128 + r * 16) = make_uint4(0, 0, 0, 0);
  }
  fence_proxy_async();
}

// d[128][n] = A B^T over the D channels, both tiles K-major in shared memory.
template <typename T, int Boxes, int ARows, int BRows>
__device__ __forceinline__ void product(uint32_t d, uint32_t A, uint32_t B, int D, int n,
                                        bool negate, uint32_t leader) {
  const uint32_t instr = instruction<T>(n, false, negate);
  const uint64_t a = operand(A, 0), b = operand(B, 0);
#pragma unroll
  for (int c = 0; c < Boxes * 4; ++c)
    if (c * 16 < D)
      mma_ss(d, a + ((c / 4) * ARows * 128 + (c % 4) * 32) / 16,
             b + ((c / 4) * BRows * 128 + (c % 4) * 32) / 16, instr, c > 0, leader);
}
// d[128][n] (+)= P X over `rows` rows (rounded up to 16) of X, a tile of BRows
// rows; P 16-bit values in tensor memory, 64 rows of X in 32 columns, the
// next 64 from 64 columns on; `gap` columns between the first 32 rows' and the
// next 32's.
template <int BRows>
__device__ __forceinline__ void accumulate(uint32_t d, uint32_t P, uint32_t X, int rows,
                                           uint32_t instr, bool add, uint32_t leader,
                                           uint32_t gap = 0) {
  const uint64_t x = operand(X, BRows * 128);
#pragma unroll
  for (int c = 0; c < BRows / 16; ++c)
    if (c * 16 < rows)
      mma_ts(d, P + c / 4 * 64 + c % 4 * 8 + (c == 2 || c == 3 ? gap : 0), x + c * 2048 / 16, instr,
             add || c > 0, leader);
}
// d[128][16] (+)= the row sums of P over `rows` columns, the same in all 16: a
// product with 16 x 16 ones, 512 bytes of them at `ones` (no swizzle: 128-byte
// blocks of 8 x 8, their order of no matter). As rounded for the product beside it.
struct Ones {
  alignas(128) uint4 x[32];
};
template <typename T>
__device__ __forceinline__ void fill_ones(Ones& ones, int t) {  // threads 0 to 31
  const uint32_t one = Elem<T>::pack(1.f, 1.f);
  ones.x[t] = make_uint4(one, one, one, one);
  fence_proxy_async();
}
template <typename T, int BRows>
__device__ __forceinline__ void row_sums(uint32_t d, uint32_t P, uint32_t ones, int rows, bool add,
                                         uint32_t leader, uint32_t gap = 0) {
  const uint64_t x = (uint64_t)((ones >> 4) & 0x3fff) | (uint64_t)(128 >> 4) << 16 |
                     (uint64_t)(256 >> 4) << 32 | (uint64_t)1 << 46;
  const uint32_t instr = instruction<T>(16, false, false);
#pragma unroll
  for (int c = 0; c < BRows / 16; ++c)
    if (c * 16 < rows)
      mma_ts(d, P + c / 4 * 64 + c % 4 * 8 + (c == 2 || c == 3 ? gap : 0), x, instr, add || c > 0,
             leader);
}

// The block's rows of no event: zeros, in 16-byte vectors, by n threads.
template <typename T, int BM>
__device__ __forceinline__ void zero_dead_rows(const FstRows& out, const RowTile& t, int h, int D,
                                               int n) {  // threads 0 to n - 1
  if (t.i0 + BM <= t.len) return;
  const int first = max(t.i0, t.len), rows = min(t.i0 + BM, t.lim) - first;
  for (int e = threadIdx.x; e < rows * (D / 8); e += n)
    *(uint4*)(row_ptr<T>(out, t, h, first + e / (D / 8)) + e % (D / 8) * 8) =
        make_uint4(0, 0, 0, 0);
}

// 16 channels, as one 32-byte store where the row lies on 32 bytes: a thread
// writes whole sectors then, which the 32 rows of a warp's store touch one
// each (two 16-byte stores pass every sector to L2 twice).
__device__ __forceinline__ void store16(void* dst, const uint32_t (&w)[8]) {
  if (((uintptr_t)dst & 31) == 0) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(w[0]),
                 "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
  } else {
    ((uint4*)dst)[0] = make_uint4(w[0], w[1], w[2], w[3]);
    ((uint4*)dst)[1] = make_uint4(w[4], w[5], w[6], w[7]);
  }
}
// A thread's row of D accumulator columns, times f, rounded and stored (whole
// warps; out may be null). `Low`: what that rounding leaves over, instead;
// `Both`: that too, to `low` (may be null), in one pass over the accumulator.
template <typename T, bool Low = false, bool Both = false>
__device__ __forceinline__ void store_row(T* out, uint32_t acc, int D, float f,
                                          T* low = nullptr) {
  for (int d = 0; d < D; d += 32) {
    float o[32];
    tmem_ld32(o, acc + d);
    tmem_wait_ld();
    pin(o);
#pragma unroll
    for (int e = 0; e < 32; e += 16) {
      if (!out || d + e >= D) break;
      auto put = [&](T* dst, const uint32_t (&w)[8]) {
        if (d + e + 16 <= D)
          store16(dst + d + e, w);
        else
          *(uint4*)(dst + d + e) = make_uint4(w[0], w[1], w[2], w[3]);
      };
      uint32_t w[8], r[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = o[e + 2 * i] * f, y = o[e + 2 * i + 1] * f;
        w[i] = Elem<T>::pack(x, y);
        if (Low || Both) r[i] = Elem<T>::pack(x - Elem<T>::lo(w[i]), y - Elem<T>::hi(w[i]));
      }
      put(out, Low ? r : w);
      if (Both && low) put(low, r);
    }
    __syncwarp();  // tcgen05.ld takes the whole warp
  }
}

// The same of up to 64 columns, less the row c (16-bit pairs, held in registers from
// before the accumulator is done) times the value in column `sum_at`.
template <typename T>
__device__ __forceinline__ void store_row_less(T* out, uint32_t acc, int D, float f,
                                               const uint32_t (&c)[32], uint32_t sum_at) {
  float sum = tmem_ld1(sum_at);
#pragma unroll
  for (int d = 0; d < 64; d += 32) {
    if (d < D) {
      float o[32];
      tmem_ld32(o, acc + d);
      tmem_wait_ld();
      pin(o);
      if (d == 0) pin(sum);
#pragma unroll
      for (int e = 0; e < 32; e += 16) {
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t x = c[(d + e) / 2 + i];
          w[i] = Elem<T>::pack(fmaf(-sum, Elem<T>::lo(x), o[e + 2 * i]) * f,
                               fmaf(-sum, Elem<T>::hi(x), o[e + 2 * i + 1]) * f);
        }
        if (out && d + e + 16 <= D)
          store16(out + d + e, w);
        else if (out && d + e < D)
          *(uint4*)(out + d + e) = make_uint4(w[0], w[1], w[2], w[3]);
      }
      __syncwarp();  // tcgen05.ld takes the whole warp
    }
  }
}

// Whether a tensor lies on the 16-byte grid that TMA and the vector stores
// need (strides of axes of one entry are never used).
inline bool on_grid(const FstGroupedProblem& p, const FstRows& r, int heads) {
  auto good = [](int64_t n, int64_t stride) {
    return n <= 1 || (stride > 0 && stride % 8 == 0 && stride < (1ll << 38));
  };
  return ((uintptr_t)r.data & 15) == 0 &&
         good(p.packed ? p.total_rows : p.max_len, r.row_stride) && good(heads, r.head_stride) &&
         good(p.packed ? 1 : p.batch, r.event_stride);
}
inline bool tc_type(const FstGroupedProblem& p) { return p.dtype != FST_F32 && p.head_dim % 8 == 0; }

// ---- the feed of work --------------------------------------------------------
//
// A block stays on its SM and works through many positions of the grid. The
// warp that feeds it asks the hardware for the next block that has not begun
// (cluster launch control cancels that block's launch and returns its index),
// looks its rows up in the work list, and hands them to the other warps
// through two slots of shared memory, while those are still busy with the
// positions before: the search, the launch and the first loads cost nothing
// then, and the grid's order (heavy blocks first) and its balance are kept.

struct Item {
  RowTile t;
  int h, kh;
  int tiles;  // of the other side; 0: only rows of no event; below 0: the end
  int whole;  // the first of them, whose keys all rows see
  int end;    // keys the block's rows see
  bool dead;  // some rows belong to no event
  int64_t out_at, stat_at;  // elements: the output's row i0, its statistics
};

struct Feed {
  alignas(16) uint4 answer;
  Item item[2];
  uint64_t full[2], empty[2], asked;
};

// One thread, before the block's barrier. `readers`: warps that take items.
__device__ __forceinline__ void feed_init(Feed& f, int readers) {
  for (int i = 0; i < 2; ++i) {
    mbar_init(smem_addr(&f.full[i]), 1);
    mbar_init(smem_addr(&f.empty[i]), readers);
  }
  mbar_init(smem_addr(&f.asked), 1);
}
// Asks for another block's place, in the feeding warp's one thread.
__device__ __forceinline__ void feed_ask(Feed& f) {
  const uint32_t bar = smem_addr(&f.asked);
  fence_proxy_async();  // the last answer has been read
  mbar_arrive_tx(bar, 16);
  asm volatile(
      "clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128"
      " [%0], [%1];" ::"r"(smem_addr(&f.answer)),
      "r"(bar)
      : "memory");
}
// The answer to question number `round`: a block's index, or -1 (none is left;
// nothing may be asked after that).
__device__ __forceinline__ int feed_answer(Feed& f, int round) {
  if (!mbar_wait(smem_addr(&f.asked), round & 1)) return -1;
  int granted, x;
  asm volatile(
      "{\n .reg .b128 r;\n .reg .pred p;\n ld.shared.b128 r, [%2];\n"
      " clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n"
      " selp.s32 %0, 1, 0, p;\n mov.s32 %1, 0;\n"
      " @p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, r;\n}"
      : "=r"(granted), "=r"(x)
      : "r"(smem_addr(&f.answer))
      : "memory");
  __syncwarp();  // read by all lanes before one of them asks again
  return granted ? x : -1;
}
// A wait that may last as long as an item of `tiles` tiles takes.
__device__ __forceinline__ bool wait_item(uint32_t bar, uint32_t parity, int tiles) {
  for (int i = 0; i <= tiles / 1024; ++i)
    if (mbar_wait(bar, parity)) return true;
  return false;
}
// Hands over item number c (whole feeding warp); `tiles`: most tiles so far.
__device__ __forceinline__ bool feed_put(Feed& f, int c, const Item& item, int tiles, int lane) {
  if (c >= 2 && !wait_item(smem_addr(&f.empty[c % 2]), (c / 2 - 1) & 1, tiles)) return false;
  if (lane == 0) {
    f.item[c % 2] = item;
    mbar_arrive(smem_addr(&f.full[c % 2]));
  }
  __syncwarp();
  return true;
}
// Takes item number c (whole warps); false at the end.
__device__ __forceinline__ bool feed_take(Feed& f, int c, Item& item, int lane) {
  if (!mbar_wait(smem_addr(&f.full[c % 2]), (c / 2) & 1)) return false;
  item = f.item[c % 2];
  __syncwarp();
  if (lane == 0) mbar_arrive(smem_addr(&f.empty[c % 2]));
  return item.tiles >= 0;
}

// Head and work-list position of a block: key heads outermost (their K and V
// stay in L2), the query heads of a group innermost (they share them).
struct BlockAt {
  int kh, h, id;
};
__device__ __forceinline__ BlockAt block_at(const FstGroupedProblem& p, int blocks, int index) {
  const int group = p.heads / p.kv_heads;
  BlockAt b;
  const int x = index / group;
  b.kh = x / blocks;
  b.id = x - b.kh * blocks;
  b.h = b.kh * group + (index - x * group);
  return b;
}

}  // namespace grouped
}  // namespace fst
