// Rotary positions: rotates the first 2 * pairs channels of every row of q and
// k by position * freqs[pair], in one launch.
//
// One read and one write of every element is all it moves, so HBM is the
// bound; the rest keeps the instructions per element few. A thread owns one
// slot (32 bytes) of a row and walks its heads: the cosines and sines of the
// slot's pairs are formed once per row, shared by the block through shared
// memory, and stay in the thread's registers for all heads. The first heads'
// loads are issued before the angles are formed.
//
// The angle is position * freq, which for far positions reaches 1e6 rad and
// more: fp32 would lose its phase. It is taken in turns in fp64,
// t = position * (freq / 2 pi), reduced exactly by t - rint(t), and the
// remainder (at most half a turn) is rounded to fp32 for sincospif. Both
// products and 1 / 2 pi round, so the angle is off by at most 2^-25 + 3 * 2^-53 |t|
// turns: 2e-7 rad up to about 2^26 turns (position 4e8 at freq 1), 4e-6 at 2^32,
// and the phase is lost from 2^50 on, as in any fp64 product. (With 1 / 2 pi in two
// parts and the products' roundings kept, exact up to position 2^53, the kernel
// spills more: 76.6 -> 79.5 us for far prompts, 24.7 -> 26.9 for padded fp32.)

#include <cuda_runtime.h>

#include <cstdint>

#include "fst_common.cuh"
#include "fst_internal.h"
#include "fst_tc_common.cuh"

namespace fst {
namespace {

constexpr int kThreads = 256;
// Measured at [21020, 32 + 8, 128] bf16, half layout, with 2 heads in flight and
// 10 heads a thread, four blocks an SM: 77 us, 5.6 TB/s (4 in flight and 4 a
// thread, three blocks: 91 us; 1 and 10, six blocks: 98 us). Chosen on that
// shape alone; at four blocks' 64 registers the vector variants spill some
// (16-bit 32 bytes, fp32 16), and interleaved 16-bit rows run at 3.9 TB/s.
constexpr int kHeads = 2;         // heads of a thread in flight
constexpr int kWalk = 10;         // heads of a thread
constexpr int kMaxRows = 32;      // rows per block
constexpr int kMaxTable = 2048;   // (cos, sin) pairs in shared memory

// V channels as they are loaded and stored: 16 bytes, kept packed until they
// are rotated, or one element.
template <typename T, int V>
struct Vec {
  uint4 w;
};
template <typename T>
struct Vec<T, 1> {
  T w;
};

// A slot is two vectors of V channels, `a` and `b`: in a rotated slot of the
// half layout the two halves of V pairs; else 2 V consecutive channels (b may
// fall behind the head's end).
struct Slot {
  int a, b;      // first channels
  int pair;      // first pair, or -1: copied
  bool has_b;
};

template <int V, bool Interleaved>
__device__ __forceinline__ Slot slot_at(const FstRotaryArgs& p, int s) {
  Slot t;
  const int rotated = Interleaved ? (2 * p.pairs + 2 * V - 1) / (2 * V) : p.pairs / V;
  if (!Interleaved && s < rotated) {
    t.a = s * V;
    t.b = p.pairs + s * V;
    t.pair = s * V;
  } else {
    t.a = Interleaved ? s * 2 * V : 2 * p.pairs + (s - rotated) * 2 * V;
    t.b = t.a + V;
    t.pair = s < rotated ? t.a / 2 : -1;
  }
  t.has_b = t.b < p.head_dim;
  return t;
}

template <typename T>
__device__ __forceinline__ float2 unpack(uint32_t w) {
  return make_float2(tc::Elem<T>::lo(w), tc::Elem<T>::hi(w));
}
__device__ __forceinline__ float2 turn(float x, float y, float2 cs) {
  return make_float2(x * cs.x - y * cs.y, y * cs.x + x * cs.y);
}

// Rotates a slot by cs, the cosines and sines of its V pairs: channel e of `a`
// with channel e of `b`, or (Adjacent) neighbours within a and then b, up to
// `left` pairs (an interleaved slot may reach past the rotated part).
template <typename T, int V, bool Adjacent>
__device__ __forceinline__ void rotate(const float2 (&cs)[V], int left, Vec<T, V>& a,
                                       Vec<T, V>& b) {
  if constexpr (V == 1) {
    const float2 r = turn(to_f<T>(a.w), to_f<T>(b.w), cs[0]);
    a.w = from_f<T>(r.x);
    b.w = from_f<T>(r.y);
  } else {
    uint32_t* wa = &a.w.x;
    uint32_t* wb = &b.w.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (Adjacent && sizeof(T) == 2) {
        const float2 x = unpack<T>(wa[i]), y = unpack<T>(wb[i]);
        const float2 u = turn(x.x, x.y, cs[i]), v = turn(y.x, y.y, cs[4 + i]);
        if (i < left) wa[i] = tc::Elem<T>::pack(u.x, u.y);
        if (4 + i < left) wb[i] = tc::Elem<T>::pack(v.x, v.y);
      } else if constexpr (Adjacent) {
        uint32_t* w = i < 2 ? wa : wb;
        const int n = i % 2 * 2;
        const float2 u = turn(__uint_as_float(w[n]), __uint_as_float(w[n + 1]), cs[i]);
        if (i < left) {
          w[n] = __float_as_uint(u.x);
          w[n + 1] = __float_as_uint(u.y);
        }
      } else if constexpr (sizeof(T) == 2) {
        const float2 x = unpack<T>(wa[i]), y = unpack<T>(wb[i]);
        const float2 u = turn(x.x, y.x, cs[2 * i]), v = turn(x.y, y.y, cs[2 * i + 1]);
        wa[i] = tc::Elem<T>::pack(u.x, v.x);
        wb[i] = tc::Elem<T>::pack(u.y, v.y);
      } else {
        const float2 u = turn(__uint_as_float(wa[i]), __uint_as_float(wb[i]), cs[i]);
        wa[i] = __float_as_uint(u.x);
        wb[i] = __float_as_uint(u.y);
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

// How a block's threads share its rows: thread u is slot u % slots, head group
// u / slots % groups, row u / slots / groups, and takes every groups-th head.
struct Shape {
  int rows, groups, heads, slots;
};

// Events: positions come from cu_seqlens, so rows may belong to no event. Those
// keep their bits: an infinity or NaN would not survive x * 1 - y * 0. (A variant
// of its own: asked of padded fp32 rows, the question costs 4 %, in spills.)
template <typename T, int V, bool Interleaved, bool Events>
__global__ void __launch_bounds__(kThreads, 4) rotary_kernel(FstRotaryArgs p, Shape sh) {
  __shared__ float2 table[kMaxTable];
  __shared__ double pos[kMaxRows];
  __shared__ int live[kMaxRows];
  const int64_t row0 = (int64_t)blockIdx.x * sh.rows;
  const int rows = (int)min((int64_t)sh.rows, p.total_rows - row0);
  // Padded: event and row of the block's first row.
  const int64_t ev0 = p.packed ? 0 : row0 / p.max_len;
  const int64_t i0 = p.packed ? row0 : row0 - ev0 * p.max_len;
  using W = Vec<T, V>;
  const int units = rows * sh.groups * sh.slots;
  bool formed = false;
  for (int u0 = 0; u0 < units; u0 += kThreads) {
    const int u = u0 + threadIdx.x, gr = u / sh.slots, r = gr / sh.groups;
    const int g = gr - r * sh.groups;
    const bool mine = u < units;
    Slot t = slot_at<V, Interleaved>(p, u - gr * sh.slots);
    int64_t ev = ev0, i = i0 + r;
    while (mine && !p.packed && i >= p.max_len) {
      i -= p.max_len;
      ++ev;
    }
    const T* q = (const T*)p.q.data + ev * p.q.event_stride + i * p.q.row_stride;
    const T* k = (const T*)p.k.data + ev * p.k.event_stride + i * p.k.row_stride;
    T* q_out = (T*)p.q_out.data + ev * p.q_out.event_stride + i * p.q_out.row_stride;
    T* k_out = (T*)p.k_out.data + ev * p.k_out.event_stride + i * p.k_out.row_stride;
    W a[kHeads], b[kHeads];
    float2 cs[V];
    for (int h0 = g; h0 < sh.heads || !formed; h0 += kHeads * sh.groups) {
#pragma unroll
      for (int n = 0; n < kHeads; ++n) {
        const int h = h0 + n * sh.groups;
        if (!mine || h >= sh.heads) continue;
        const T* src = h < p.heads ? q + h * p.q.head_stride
                                   : k + (h - p.heads) * p.k.head_stride;
        a[n] = *(const W*)(src + t.a);
        if (t.has_b) b[n] = *(const W*)(src + t.b);
      }
      if (!formed) {
        // The angles, while the loads are on their way.
        formed = true;
        if (threadIdx.x < rows) {
          const int64_t at = row0 + threadIdx.x;
          int64_t count = 0;
          live[threadIdx.x] =
              position_of(p, at, p.packed ? at : (i0 + threadIdx.x) % p.max_len, count);
          pos[threadIdx.x] = (double)count;
        }
        __syncthreads();
        for (int e = threadIdx.x; e < rows * p.pairs; e += kThreads) {
          const int er = e / p.pairs;
          float sn = 0.f, c = 1.f;
          if (live[er]) {
            const double turns = pos[er] * (p.freqs[e - er * p.pairs] * 0.15915494309189533577);
            sincospif((float)(2.0 * (turns - rint(turns))), &sn, &c);
            sn *= p.inverse ? -p.magnitude : p.magnitude;
            c *= p.magnitude;
          }
          table[e] = make_float2(c, sn);
        }
        __syncthreads();
      }
      if (!mine) continue;
      if (Events && h0 == g && !live[r]) t.pair = -1;
      if (h0 == g && t.pair >= 0) {
#pragma unroll
        for (int e = 0; e < V; ++e)
          cs[e] = t.pair + e < p.pairs ? table[r * p.pairs + t.pair + e] : make_float2(1.f, 0.f);
      }
#pragma unroll
      for (int n = 0; n < kHeads; ++n) {
        const int h = h0 + n * sh.groups;
        if (h >= sh.heads) continue;
        if (t.pair >= 0) rotate<T, V, Interleaved && V != 1>(cs, p.pairs - t.pair, a[n], b[n]);
        T* dst = h < p.heads ? q_out + h * p.q_out.head_stride
                             : k_out + (h - p.heads) * p.k_out.head_stride;
        *(W*)(dst + t.a) = a[n];
        if (t.has_b) *(W*)(dst + t.b) = b[n];
      }
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
  // kWalk heads a thread where there are as many, and as many rows as fill
  // the block.
  int groups = (heads + kWalk - 1) / kWalk;
  if (groups * (int64_t)slots > kThreads) groups = slots < kThreads ? kThreads / slots : 1;
  int rows = kThreads / (groups * slots);
  if (rows > kMaxRows) rows = kMaxRows;
  if (p.pairs > 0 && rows > kMaxTable / p.pairs) rows = kMaxTable / p.pairs;
  if (rows < 1) rows = 1;
  const int64_t blocks = (p.total_rows + rows - 1) / rows;
  if (blocks >= (1ll << 31))
    return api_fail(FST_ERR_UNSUPPORTED, "rotary: %lld rows are too many",
                    (long long)p.total_rows);
  const Shape sh{rows, groups, heads, slots};
  const bool events = p.packed && !p.positions;
  const auto kernel =
      vec ? (p.interleaved ? (events ? rotary_kernel<T, V, true, true> : rotary_kernel<T, V, true, false>)
                           : (events ? rotary_kernel<T, V, false, true> : rotary_kernel<T, V, false, false>))
          : (p.interleaved ? (events ? rotary_kernel<T, 1, true, true> : rotary_kernel<T, 1, true, false>)
                           : (events ? rotary_kernel<T, 1, false, true> : rotary_kernel<T, 1, false, false>));
  kernel<<<(unsigned)blocks, kThreads, 0, st>>>(p, sh);
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
