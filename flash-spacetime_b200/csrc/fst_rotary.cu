// Rotary positions: rotates the first 2 * pairs channels of every row of q and
// k by position * freqs[pair], in one launch.
//
// One read and one write of every element is all it moves, so HBM is the
// bound; the rest is arranged around that. A block takes a few rows (about
// four 32-byte slots per thread) with all their heads, so the angles are
// formed once per row and pair and shared by the heads through shared memory;
// each thread issues its loads before the angles are formed.
//
// The angle is position * freq, which for far positions reaches 1e6 rad and
// more: fp32 would lose its phase. It is taken in turns in fp64,
// t = position * (freq / 2 pi), reduced exactly by t - rint(t), and only the
// remainder (at most half a turn) is rounded to fp32 for sincospif: 2^-25
// turns, 2e-7 rad, whatever the position.

#include <cuda_runtime.h>

#include <cstdint>

#include "fst_common.cuh"
#include "fst_internal.h"

namespace fst {
namespace {

constexpr int kThreads = 256;
constexpr int kItems = 4;         // slots per thread and pass
constexpr int kMaxRows = 16;      // rows per block
constexpr int kMaxTable = 2048;   // (cos, sin) pairs in shared memory

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T x[V];
};

// A slot is two vectors of V channels, `a` and `b`: in a rotated slot of the
// half layout the two halves of V pairs; else 2 V consecutive channels (b may
// fall behind the head's end).
struct Slot {
  int a, b;      // first channels
  int pair;      // first pair, or -1: copied
  bool has_b;
};

template <int V>
__device__ __forceinline__ Slot slot_at(const FstRotaryArgs& p, int s) {
  Slot t;
  const int rotated = p.interleaved ? (2 * p.pairs + 2 * V - 1) / (2 * V) : p.pairs / V;
  if (!p.interleaved && s < rotated) {
    t.a = s * V;
    t.b = p.pairs + s * V;
    t.pair = s * V;
  } else {
    t.a = p.interleaved ? s * 2 * V : 2 * p.pairs + (s - rotated) * 2 * V;
    t.b = t.a + V;
    t.pair = s < rotated ? t.a / 2 : -1;
  }
  t.has_b = t.b < p.head_dim;
  return t;
}

template <typename T, int V>
__device__ __forceinline__ void rotate(const FstRotaryArgs& p, const Slot& t, const float2* cs,
                                       Vec<T, V>& a, Vec<T, V>& b) {
  if (t.pair < 0) return;
  if (!p.interleaved || V == 1) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float2 c = cs[t.pair + e];
      const float x = to_f<T>(a.x[e]), y = to_f<T>(b.x[e]);
      a.x[e] = from_f<T>(x * c.x - y * c.y);
      b.x[e] = from_f<T>(y * c.x + x * c.y);
    }
  } else {
    // Pairs lie inside the vectors; the slot may reach past the rotated part.
#pragma unroll
    for (int e = 0; e + 1 < V; e += 2) {
      const int pa = t.pair + e / 2, pb = pa + V / 2;
      if (pa < p.pairs) {
        const float2 c = cs[pa];
        const float x = to_f<T>(a.x[e]), y = to_f<T>(a.x[e + 1]);
        a.x[e] = from_f<T>(x * c.x - y * c.y);
        a.x[e + 1] = from_f<T>(y * c.x + x * c.y);
      }
      if (pb < p.pairs) {
        const float2 c = cs[pb];
        const float x = to_f<T>(b.x[e]), y = to_f<T>(b.x[e + 1]);
        b.x[e] = from_f<T>(x * c.x - y * c.y);
        b.x[e + 1] = from_f<T>(y * c.x + x * c.y);
      }
    }
  }
}

// Position of flat row `row` ((ev, i) when padded); false: a packed row of no
// event.
__device__ __forceinline__ bool position_of(const FstRotaryArgs& p, int64_t row, int64_t i,
                                            int64_t& pos) {
  if (p.positions) {
    pos = p.positions_64 ? ((const int64_t*)p.positions)[row] : ((const int32_t*)p.positions)[row];
    return true;
  }
  pos = i;
  if (!p.packed) return true;
  if (p.batch <= 0 || row < p.cu_seqlens[0] || row >= p.cu_seqlens[p.batch]) return false;
  int lo = 0, hi = p.batch;  // cu[lo] <= row < cu[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (p.cu_seqlens[mid] <= row)
      lo = mid;
    else
      hi = mid;
  }
  pos = row - p.cu_seqlens[lo];
  return true;
}

// Quotients of a block's item numbers: n / d = umulhi(n, ceil(2^32 / d)) while
// n d < 2^32, which the host makes sure of (a 32-bit division would cost more
// instructions than the rotation).
struct Split {
  int rows_per_block, heads, slots;
  uint32_t by_heads, by_slots;  // 0: the divisor is 1
};
__device__ __forceinline__ int quotient(int n, uint32_t by) {
  return by ? (int)__umulhi((uint32_t)n, by) : n;
}

template <typename T, int V>
__global__ void __launch_bounds__(kThreads, 3) rotary_kernel(FstRotaryArgs p, Split sp) {
  __shared__ float2 cs[kMaxTable];
  __shared__ double pos[kMaxRows];
  __shared__ int live[kMaxRows];
  const int64_t row0 = (int64_t)blockIdx.x * sp.rows_per_block;
  const int rows = (int)min((int64_t)sp.rows_per_block, p.total_rows - row0);
  // Padded: event and row of the block's first row.
  const int64_t ev0 = p.packed ? 0 : row0 / p.max_len;
  const int64_t i0 = p.packed ? row0 : row0 - ev0 * p.max_len;
  using W = Vec<T, V>;
  const int items = rows * sp.heads * sp.slots;  // host: below 2^31
  for (int base = 0; base < items; base += kThreads * kItems) {
    W a[kItems], b[kItems];
    T* dst[kItems];
    int where[kItems];  // row of the block and slot of the head
#pragma unroll
    for (int n = 0; n < kItems; ++n) {
      const int item = base + n * kThreads + threadIdx.x;
      dst[n] = nullptr;
      if (item >= items) continue;
      const int rh = quotient(item, sp.by_slots), s = item - rh * sp.slots;
      const int r = quotient(rh, sp.by_heads), h = rh - r * sp.heads;
      where[n] = r << 16 | s;  // slots: at most 1024 / 2 + 1
      const Slot t = slot_at<V>(p, s);
      int64_t ev = ev0, i = i0 + r;
      while (!p.packed && i >= p.max_len) {
        i -= p.max_len;
        ++ev;
      }
      const bool is_k = h >= p.heads;
      const FstRows& in = is_k ? p.k : p.q;
      const FstRows& out = is_k ? p.k_out : p.q_out;
      const int hh = is_k ? h - p.heads : h;
      const T* src =
          (const T*)in.data + ev * in.event_stride + i * in.row_stride + hh * in.head_stride;
      dst[n] = (T*)out.data + ev * out.event_stride + i * out.row_stride + hh * out.head_stride;
      a[n] = *(const W*)(src + t.a);
      if (t.has_b) b[n] = *(const W*)(src + t.b);
    }
    if (base == 0) {
      // The angles, while the loads are on their way.
      if (threadIdx.x < rows) {
        const int64_t at = row0 + threadIdx.x;
        int64_t count = 0;
        live[threadIdx.x] =
            position_of(p, at, p.packed ? at : (i0 + threadIdx.x) % p.max_len, count);
        pos[threadIdx.x] = (double)count;
      }
      __syncthreads();
      for (int e = threadIdx.x; e < rows * p.pairs; e += kThreads) {
        const int r = e / p.pairs;
        float sn = 0.f, c = 1.f;
        if (live[r]) {
          const double t = pos[r] * (p.freqs[e - r * p.pairs] * 0.15915494309189533577);
          sincospif((float)(2.0 * (t - rint(t))), &sn, &c);
          sn *= p.inverse ? -p.magnitude : p.magnitude;
          c *= p.magnitude;
        }
        cs[e] = make_float2(c, sn);
      }
      __syncthreads();
    }
#pragma unroll
    for (int n = 0; n < kItems; ++n) {
      if (!dst[n]) continue;
      const Slot t = slot_at<V>(p, where[n] & 0xffff);
      rotate<T, V>(p, t, cs + (where[n] >> 16) * p.pairs, a[n], b[n]);
      *(W*)(dst[n] + t.a) = a[n];
      if (t.has_b) *(W*)(dst[n] + t.b) = b[n];
    }
  }
}

bool vector_ok(const FstRows& r, int v) {
  return ((uintptr_t)r.data & 15) == 0 && r.event_stride % v == 0 && r.head_stride % v == 0 &&
         r.row_stride % v == 0;
}

template <typename T>
int launch(const FstRotaryArgs& p, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  // 16-byte vectors where every row starts on 16 bytes and neither the head
  // nor (half layout) its rotated halves end inside a vector; else elements.
  const bool vec = p.head_dim % V == 0 && (p.interleaved || p.pairs % V == 0) &&
                   vector_ok(p.q, V) && vector_ok(p.q_out, V) &&
                   (!p.k.data || (vector_ok(p.k, V) && vector_ok(p.k_out, V)));
  const int w = vec ? V : 1;
  const int rot = p.interleaved ? (2 * p.pairs + 2 * w - 1) / (2 * w) : p.pairs / w;
  const int slots = p.interleaved ? (p.head_dim + 2 * w - 1) / (2 * w)
                                  : rot + (p.head_dim - 2 * p.pairs + 2 * w - 1) / (2 * w);
  const int heads = p.heads + (p.k.data ? p.kv_heads : 0);
  const int64_t row_items = (int64_t)heads * slots;
  int64_t rows = kThreads * kItems / row_items;
  if (rows > kMaxRows) rows = kMaxRows;
  if (p.pairs > 0 && rows > kMaxTable / p.pairs) rows = kMaxTable / p.pairs;
  if (rows < 1) rows = 1;
  if (row_items >= (1ll << 31) ||
      rows * row_items * (heads > slots ? heads : slots) >= (1ll << 32))
    return api_fail(FST_ERR_UNSUPPORTED, "rotary: %d heads of %d are too many", heads, p.head_dim);
  const int64_t blocks = (p.total_rows + rows - 1) / rows;
  if (blocks >= (1ll << 31))
    return api_fail(FST_ERR_UNSUPPORTED, "rotary: %lld rows are too many",
                    (long long)p.total_rows);
  auto by = [](int d) { return d > 1 ? (uint32_t)(((1ull << 32) + d - 1) / d) : 0u; };
  const Split sp{(int)rows, heads, slots, by(heads), by(slots)};
  if (vec)
    rotary_kernel<T, V><<<(unsigned)blocks, kThreads, 0, st>>>(p, sp);
  else
    rotary_kernel<T, 1><<<(unsigned)blocks, kThreads, 0, st>>>(p, sp);
  count_launch();
  return FST_OK;
}

}  // namespace

int launch_rotary(const FstRotaryArgs& p, cudaStream_t st) {
  if (p.dtype == FST_F32) return launch<float>(p, st);
  if (p.dtype == FST_BF16) return launch<__nv_bfloat16>(p, st);
  return launch<__half>(p, st);
}

}  // namespace fst
