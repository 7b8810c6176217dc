// Grouped-head attention: addressing and the work list shared by its CUDA-core
// and tensor-core kernels.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "fst_common.cuh"
#include "fst_internal.h"

namespace fst {
namespace grouped {

// One block's rows of one event. Rows i0 <= i < min(i0 + BM, lim) belong to
// the block: those below len are live, the others are rows of no event, whose
// outputs are written 0.
struct RowTile {
  int ev;    // event index of the padded layout, 0 when packed
  int base;  // buffer row of the event's row 0
  int len;   // live rows of the event
  int lim;   // rows the event (or the gap between events) covers
  int i0;    // first row of the block
};

// Blocks of bm rows that the work list of `p` needs per head. Packed: event e
// starts at list position cu[e] / bm + e + 1, which leaves every event at
// least ceil(len / bm) positions (floor(b) - floor(a) + 1 >= ceil(b - a)), so
// the list needs no prefix pass and no host synchronisation; the gap before
// the first event and the one behind the last are entries -1 and B.
__host__ __device__ __forceinline__ int64_t list_blocks(const FstGroupedProblem& p, int bm) {
  if (p.packed) return p.total_rows / bm + p.batch + 2;
  return (int64_t)p.batch * ((p.max_len + bm - 1) / bm);
}

__device__ __forceinline__ int clamp_row(int x, int64_t n) {
  return x < 0 ? 0 : (x > n ? (int)n : x);
}
// Buffer row at which entry e of the packed list starts (e = -1 .. B + 1).
// Clamped, so offsets that are wrong never lead out of the tensors.
__device__ __forceinline__ int entry_row(const FstGroupedProblem& p, int e) {
  if (e < 0) return 0;
  if (e > p.batch) return (int)p.total_rows;
  return clamp_row(__ldg(p.cu_seqlens + e), p.total_rows);
}

// Block `id` of the list (called by whole warps). `reverse`: an event's live
// blocks last rows first, which puts the causal ones with most keys at the
// front. Returns false when the position is empty.
template <int BM>
__device__ __forceinline__ bool find_tile(const FstGroupedProblem& p, int id, bool reverse,
                                          RowTile& t) {
  int tile, live;
  if (!p.packed) {
    const int per = (p.max_len + BM - 1) / BM;
    t.ev = id / per;
    tile = id - t.ev * per;
    t.base = 0;
    t.len = clamp_row(__ldg(p.seqlens + t.ev), p.max_len);
    t.lim = p.max_len;
  } else {
    // Largest entry whose position is <= id: 33-way search, one probe a lane.
    // The rows at both ends of the range are kept, so that each step is the
    // only trip to memory: one up to 31 events, two up to 1055.
    const int lane = threadIdx.x & 31;
    int lo = -1, hi = p.batch + 1, a = 0, b = (int)p.total_rows;
    while (hi - lo > 1) {
      const int step = (hi - lo + 32) / 33;
      const int e = lo + step * (lane + 1);
      const int row = e < hi ? entry_row(p, e) : b;
      const bool at = e < hi && row / BM + e + 1 <= id;
      const int first = __ffs(~__ballot_sync(0xffffffffu, at)) - 1;
      const int n = first < 0 ? 32 : first;  // probes at or below id
      const int below = __shfl_sync(0xffffffffu, row, n > 0 ? n - 1 : 0);
      const int above = __shfl_sync(0xffffffffu, row, n < 32 ? n : 31);
      a = n > 0 ? below : a;
      b = n < 32 ? above : b;
      lo += step * n;
      hi = min(hi, lo + step);
    }
    t.ev = 0;
    t.base = a;
    t.lim = max(b - a, 0);
    t.len = (lo >= 0 && lo < p.batch) ? t.lim : 0;
    tile = id - (a / BM + lo + 1);
  }
  live = (t.len + BM - 1) / BM;
  if (reverse && tile < live) tile = live - 1 - tile;
  // A position behind the entry's last block is empty (compared before tile is
  // multiplied: positions of other entries' blocks may lie far behind).
  if (tile >= (t.lim + BM - 1) / BM) return false;
  t.i0 = tile * BM;
  return true;
}

template <typename T>
__device__ __forceinline__ T* row_ptr(const FstRows& r, const RowTile& t, int h, int i) {
  return (T*)r.data + (int64_t)t.ev * r.event_stride + (int64_t)h * r.head_stride +
         (int64_t)(t.base + i) * r.row_stride;
}

// Offset of (h, row t.base + i) in a dense statistics tensor of nh heads.
__device__ __forceinline__ int64_t stat_at(const FstGroupedProblem& p, const RowTile& t, int nh,
                                           int h, int i) {
  const int64_t n = p.packed ? p.total_rows : p.max_len;
  return ((int64_t)t.ev * nh + h) * n + t.base + i;
}

// Host side (fst_grouped_simt.cu, fst_grouped_fwd.cu, fst_grouped_bwd.cu).
int simt_forward(const FstGroupedForwardArgs& a, cudaStream_t st);
int simt_backward(const FstGroupedBackwardArgs& a, cudaStream_t st);
// Whether the tensor-core kernels take a call: 16-bit, Dh a multiple of 8, and
// every tensor on the 16-byte grid that TMA and the vector stores need.
bool tc_takes(const FstGroupedForwardArgs& a);
bool tc_takes(const FstGroupedBackwardArgs& a);
int tc_forward(const FstGroupedForwardArgs& a, cudaStream_t st);
int tc_backward(const FstGroupedBackwardArgs& a, cudaStream_t st);

}  // namespace grouped
}  // namespace fst
