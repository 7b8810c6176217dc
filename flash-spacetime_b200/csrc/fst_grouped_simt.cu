// Grouped-head attention on the CUDA cores: fp32 inputs, and 16-bit ones whose
// head size or strides the tensor-core kernels do not take. All sums fp32.
//
// One block of 256 threads owns 64 rows of one event and head: query rows in
// the forward and dq kernels, key rows in the dk / dv kernel, which walks the
// 64-row tiles of the other side and, for dk / dv, the query heads of the
// group in order. Every output element has one writer and a fixed order of
// additions. Logits live in 4 x 4 register tiles (rows 4 ty + r, columns
// tx + 16 c), probabilities pass through shared memory to the second product.
//
// Softmax statistics are kept in the base-2 domain: x = scale log2(e) q.k,
// m = max x, l = sum 2^(x - m), lse = (m + log2 l) ln 2.
//
// FMA-bound: a 64 x 64 x D product reads 2 float4 per 16 FMAs.

#include <cuda_runtime.h>

#include <atomic>

#include "fst_grouped.cuh"

namespace fst {
namespace grouped {
namespace {

constexpr int kB = 64;        // tile rows and columns
constexpr int kThreads = 256;
constexpr int kPS = kB + 4;   // padded row of a probability tile

// Rows of a [64][DM + 4] tile from global memory; rows at or past n and
// channels past D are zero, so nothing behind an event's end is read.
template <typename T, int DM>
__device__ __forceinline__ void load_tile(float* dst, const T* src, int64_t stride, int n, int D) {
  for (int e = threadIdx.x; e < kB * DM; e += kThreads) {
    const int r = e / DM, d = e % DM;
    dst[r * (DM + 4) + d] = (r < n && d < D) ? to_f<T>(src[r * stride + d]) : 0.f;
  }
}

// s[r][c] = A[4 ty + r] . B[tx + 16 c]
template <int DM>
__device__ __forceinline__ void product(const float* A, const float* B, int ty, int tx,
                                        float (&s)[4][4]) {
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int c = 0; c < 4; ++c) s[r][c] = 0.f;
#pragma unroll 4
  for (int d = 0; d < DM; d += 4) {
    float4 a[4], b[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) a[r] = *(const float4*)(A + (4 * ty + r) * (DM + 4) + d);
#pragma unroll
    for (int c = 0; c < 4; ++c) b[c] = *(const float4*)(B + (tx + 16 * c) * (DM + 4) + d);
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        s[r][c] = fmaf(a[r].x, b[c].x, s[r][c]);
        s[r][c] = fmaf(a[r].y, b[c].y, s[r][c]);
        s[r][c] = fmaf(a[r].z, b[c].z, s[r][c]);
        s[r][c] = fmaf(a[r].w, b[c].w, s[r][c]);
      }
  }
}

// acc[r][c] += sum_j P[4 ty + r][j] X[j][tx + 16 c]
template <int DM>
__device__ __forceinline__ void accumulate(const float* P, const float* X, int ty, int tx,
                                           float (&acc)[4][DM / 16]) {
#pragma unroll 2
  for (int j = 0; j < kB; j += 4) {
    float4 p[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) p[r] = *(const float4*)(P + (4 * ty + r) * kPS + j);
#pragma unroll
    for (int jj = 0; jj < 4; ++jj)
#pragma unroll
      for (int c = 0; c < DM / 16; ++c) {
        const float x = X[(j + jj) * (DM + 4) + tx + 16 * c];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float pv = jj == 0 ? p[r].x : jj == 1 ? p[r].y : jj == 2 ? p[r].z : p[r].w;
          acc[r][c] = fmaf(pv, x, acc[r][c]);
        }
      }
  }
}

__device__ __forceinline__ float half_warp_max(float x) {
#pragma unroll
  for (int o = 8; o; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
  return x;
}
__device__ __forceinline__ float half_warp_sum(float x) {
#pragma unroll
  for (int o = 8; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

// Rows of no event among the block's rows of head h: written 0.
template <typename T>
__device__ __forceinline__ void zero_rows(const FstRows& out, const RowTile& t, int h, int D) {
  const int first = max(t.i0, t.len), last = min(t.i0 + kB, t.lim);
  for (int64_t e = threadIdx.x; e < (int64_t)(last - first) * D; e += kThreads)
    row_ptr<T>(out, t, h, first + (int)(e / D))[e % D] = from_f<T>(0.f);
}

template <typename T, int DM>
__device__ __forceinline__ void store_rows(const FstRows& out, const RowTile& t, int h, int D,
                                           int ty, int tx, const float (&acc)[4][DM / 16],
                                           const float (&mul)[4]) {
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int i = t.i0 + 4 * ty + r;
    if (i >= t.len) continue;
    T* o = row_ptr<T>(out, t, h, i);
#pragma unroll
    for (int c = 0; c < DM / 16; ++c)
      if (tx + 16 * c < D) o[tx + 16 * c] = from_f<T>(acc[r][c] * mul[r]);
  }
}

template <typename T, int DM>
__global__ void __launch_bounds__(kThreads) fwd_kernel(FstGroupedForwardArgs a) {
  extern __shared__ float4 smem4[];
  float* Q = (float*)smem4;
  float* K = Q + kB * (DM + 4);
  float* V = K + kB * (DM + 4);
  float* P = V + kB * (DM + 4);
  const FstGroupedProblem& p = a.prob;
  const int h = blockIdx.x % p.heads, kh = h / (p.heads / p.kv_heads);
  RowTile t;
  if (!find_tile<kB>(p, blockIdx.x / p.heads, p.causal, t)) return;
  const int D = p.head_dim, ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  zero_rows<T>(a.out, t, h, D);
  if (t.i0 >= t.len) return;
  load_tile<T, DM>(Q, row_ptr<T>(a.q, t, h, t.i0), a.q.row_stride, t.len - t.i0, D);
  const float c2 = p.scale * kLog2e;
  float acc[4][DM / 16] = {}, m[4], l[4] = {};
#pragma unroll
  for (int r = 0; r < 4; ++r) m[r] = -INFINITY;
  const int end = p.causal ? min(t.len, t.i0 + kB) : t.len;
  for (int j0 = 0; j0 < end; j0 += kB) {
    __syncthreads();
    load_tile<T, DM>(K, row_ptr<T>(a.k, t, kh, j0), a.k.row_stride, t.len - j0, D);
    load_tile<T, DM>(V, row_ptr<T>(a.v, t, kh, j0), a.v.row_stride, t.len - j0, D);
    __syncthreads();
    float s[4][4];
    product<DM>(Q, K, ty, tx, s);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = t.i0 + 4 * ty + r;
      const int last = p.causal ? min(i + 1, t.len) : t.len;  // keys below it are seen
      float mx = m[r];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        s[r][c] = j0 + tx + 16 * c < last ? s[r][c] * c2 : -INFINITY;
        mx = fmaxf(mx, s[r][c]);
      }
      mx = half_warp_max(mx);
      // A row that has seen nothing but -inf logits keeps a zero offset.
      const float off = mx == -INFINITY ? 0.f : mx;
      const float keep = exp2f(m[r] - off);
      float sum = 0.f;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        s[r][c] = exp2f(s[r][c] - off);
        sum += s[r][c];
        P[(4 * ty + r) * kPS + tx + 16 * c] = s[r][c];
      }
      l[r] = l[r] * keep + half_warp_sum(sum);
      m[r] = mx;
#pragma unroll
      for (int c = 0; c < DM / 16; ++c) acc[r][c] *= keep;
    }
    __syncwarp();  // a row of P is written and read by one half warp
    accumulate<DM>(P, V, ty, tx, acc);
  }
  float inv[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    inv[r] = 1.f / l[r];
    const int i = t.i0 + 4 * ty + r;
    if (tx == 0 && i < t.len)
      a.lse[stat_at(p, t, p.heads, h, i)] = (m[r] + log2f(l[r])) / kLog2e;
  }
  store_rows<T, DM>(a.out, t, h, D, ty, tx, acc, inv);
  if (a.out_low.data) {
    // What rounding to T left over.
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int c = 0; c < DM / 16; ++c) {
        const float x = acc[r][c] * inv[r];
        acc[r][c] = x - to_f<T>(from_f<T>(x));
      }
    const float one[4] = {1.f, 1.f, 1.f, 1.f};
    store_rows<T, DM>(a.out_low, t, h, D, ty, tx, acc, one);
  }
}

// dq, and D_i = dO_i . o_i for the dk / dv kernel.
template <typename T, int DM>
__global__ void __launch_bounds__(kThreads) dq_kernel(FstGroupedBackwardArgs a) {
  extern __shared__ float4 smem4[];
  float* Q = (float*)smem4;
  float* G = Q + kB * (DM + 4);
  float* K = G + kB * (DM + 4);
  float* V = K + kB * (DM + 4);
  float* P = V + kB * (DM + 4);
  const FstGroupedProblem& p = a.prob;
  const int h = blockIdx.x % p.heads, kh = h / (p.heads / p.kv_heads);
  RowTile t;
  if (!find_tile<kB>(p, blockIdx.x / p.heads, p.causal, t)) return;
  const int D = p.head_dim, ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  zero_rows<T>(a.dq, t, h, D);
  if (t.i0 >= t.len) return;
  load_tile<T, DM>(Q, row_ptr<T>(a.q, t, h, t.i0), a.q.row_stride, t.len - t.i0, D);
  load_tile<T, DM>(G, row_ptr<T>(a.dout, t, h, t.i0), a.dout.row_stride, t.len - t.i0, D);
  load_tile<T, DM>(K, row_ptr<T>(a.out, t, h, t.i0), a.out.row_stride, t.len - t.i0, D);
  const bool low = a.out_low.data != nullptr;
  if (low)
    load_tile<T, DM>(V, row_ptr<T>(a.out_low, t, h, t.i0), a.out_low.row_stride, t.len - t.i0, D);
  __syncthreads();
  const float c2 = p.scale * kLog2e;
  float lse2[4], delta[4], acc[4][DM / 16] = {};
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int i = t.i0 + 4 * ty + r;
    float sum = 0.f;
    for (int d = tx; d < DM; d += 16)
    {
      const int at = (4 * ty + r) * (DM + 4) + d;
      sum = fmaf(G[at], low ? K[at] + V[at] : K[at], sum);
    }
    delta[r] = half_warp_sum(sum);
    const int64_t at = stat_at(p, t, p.heads, h, i);
    lse2[r] = i < t.len ? a.lse[at] * kLog2e : 0.f;
    if (tx == 0 && i < t.len) a.stats[at] = delta[r];
  }
  const int end = p.causal ? min(t.len, t.i0 + kB) : t.len;
  for (int j0 = 0; j0 < end; j0 += kB) {
    __syncthreads();
    load_tile<T, DM>(K, row_ptr<T>(a.k, t, kh, j0), a.k.row_stride, t.len - j0, D);
    load_tile<T, DM>(V, row_ptr<T>(a.v, t, kh, j0), a.v.row_stride, t.len - j0, D);
    __syncthreads();
    float s[4][4], dp[4][4];
    product<DM>(Q, K, ty, tx, s);
    product<DM>(G, V, ty, tx, dp);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = t.i0 + 4 * ty + r;
      const int last = p.causal ? min(i + 1, t.len) : t.len;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        // A row that sees one key has P = 1 and dP = D: dS is 0, not the
        // rounding of two sums of different order.
        const bool seen = j0 + tx + 16 * c < last && last > 1;
        const float pr = exp2f(s[r][c] * c2 - lse2[r]);
        P[(4 * ty + r) * kPS + tx + 16 * c] = seen ? pr * (dp[r][c] - delta[r]) : 0.f;
      }
    }
    __syncwarp();
    accumulate<DM>(P, K, ty, tx, acc);
  }
  const float mul[4] = {p.scale, p.scale, p.scale, p.scale};
  store_rows<T, DM>(a.dq, t, h, D, ty, tx, acc, mul);
}

template <typename T, int DM>
__global__ void __launch_bounds__(kThreads) dkv_kernel(FstGroupedBackwardArgs a) {
  extern __shared__ float4 smem4[];
  float* K = (float*)smem4;
  float* V = K + kB * (DM + 4);
  float* Q = V + kB * (DM + 4);
  float* G = Q + kB * (DM + 4);
  float* P = G + kB * (DM + 4);
  float* S = P + kB * kPS;
  float* lse2 = S + kB * kPS;
  float* delta = lse2 + kB;
  const FstGroupedProblem& p = a.prob;
  const int kh = blockIdx.x % p.kv_heads, group = p.heads / p.kv_heads;
  RowTile t;
  if (!find_tile<kB>(p, blockIdx.x / p.kv_heads, false, t)) return;
  const int D = p.head_dim, ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  zero_rows<T>(a.dk, t, kh, D);
  zero_rows<T>(a.dv, t, kh, D);
  if (t.i0 >= t.len) return;
  load_tile<T, DM>(K, row_ptr<T>(a.k, t, kh, t.i0), a.k.row_stride, t.len - t.i0, D);
  load_tile<T, DM>(V, row_ptr<T>(a.v, t, kh, t.i0), a.v.row_stride, t.len - t.i0, D);
  const float c2 = p.scale * kLog2e;
  float dk[4][DM / 16] = {}, dv[4][DM / 16] = {};
  for (int h = kh * group; h < (kh + 1) * group; ++h) {
    for (int q0 = p.causal ? t.i0 : 0; q0 < t.len; q0 += kB) {
      __syncthreads();
      load_tile<T, DM>(Q, row_ptr<T>(a.q, t, h, q0), a.q.row_stride, t.len - q0, D);
      load_tile<T, DM>(G, row_ptr<T>(a.dout, t, h, q0), a.dout.row_stride, t.len - q0, D);
      if (threadIdx.x < kB) {
        const bool live = q0 + (int)threadIdx.x < t.len;
        const int64_t at = stat_at(p, t, p.heads, h, q0 + threadIdx.x);
        lse2[threadIdx.x] = live ? a.lse[at] * kLog2e : 0.f;
        delta[threadIdx.x] = live ? a.stats[at] : 0.f;
      }
      __syncthreads();
      float s[4][4], dp[4][4];  // [key row][query column]
      product<DM>(K, Q, ty, tx, s);
      product<DM>(V, G, ty, tx, dp);
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int col = tx + 16 * c, i = q0 + col;
          const bool seen = i < t.len && (!p.causal || t.i0 + 4 * ty + r <= i);
          const float pr = seen ? exp2f(s[r][c] * c2 - lse2[col]) : 0.f;
          P[(4 * ty + r) * kPS + col] = pr;
          const bool several = p.causal ? i > 0 : t.len > 1;  // row i sees more than one key
          S[(4 * ty + r) * kPS + col] = seen && several ? pr * (dp[r][c] - delta[col]) : 0.f;
        }
      __syncwarp();
      accumulate<DM>(P, G, ty, tx, dv);
      accumulate<DM>(S, Q, ty, tx, dk);
    }
  }
  const float one[4] = {1.f, 1.f, 1.f, 1.f};
  const float mul[4] = {p.scale, p.scale, p.scale, p.scale};
  store_rows<T, DM>(a.dv, t, kh, D, ty, tx, dv, one);
  store_rows<T, DM>(a.dk, t, kh, D, ty, tx, dk, mul);
}

template <typename F, typename A>
int launch(F kernel, std::atomic<uint64_t>& done, int bytes, int heads, const A& a,
           cudaStream_t st) {
  const int64_t blocks = list_blocks(a.prob, kB) * heads;
  if (blocks == 0) return FST_OK;
  const int e = allow_dynamic_smem((const void*)kernel, bytes, done);
  if (e) return api_fail(FST_ERR_CUDA, "shared memory: %s", cudaGetErrorString((cudaError_t)e));
  kernel<<<(unsigned)blocks, kThreads, bytes, st>>>(a);
  count_launch();
  return FST_OK;
}

constexpr int tile_bytes(int dm) { return kB * (dm + 4) * 4; }
constexpr int prob_bytes = kB * kPS * 4;

template <typename T, int DM>
int forward_dm(const FstGroupedForwardArgs& a, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};
  return launch(fwd_kernel<T, DM>, done, 3 * tile_bytes(DM) + prob_bytes, a.prob.heads, a, st);
}

template <typename T, int DM>
int backward_dm(const FstGroupedBackwardArgs& a, cudaStream_t st) {
  static std::atomic<uint64_t> done_q{0}, done_kv{0};
  const int rc = launch(dq_kernel<T, DM>, done_q, 4 * tile_bytes(DM) + prob_bytes, a.prob.heads,
                        a, st);
  if (rc) return rc;
  return launch(dkv_kernel<T, DM>, done_kv, 4 * tile_bytes(DM) + 2 * prob_bytes + 2 * kB * 4,
                a.prob.kv_heads, a, st);
}

template <typename T>
int forward_t(const FstGroupedForwardArgs& a, cudaStream_t st) {
  if (a.prob.head_dim <= 32) return forward_dm<T, 32>(a, st);
  if (a.prob.head_dim <= 64) return forward_dm<T, 64>(a, st);
  return forward_dm<T, 128>(a, st);
}

template <typename T>
int backward_t(const FstGroupedBackwardArgs& a, cudaStream_t st) {
  if (a.prob.head_dim <= 32) return backward_dm<T, 32>(a, st);
  if (a.prob.head_dim <= 64) return backward_dm<T, 64>(a, st);
  return backward_dm<T, 128>(a, st);
}

}  // namespace

int simt_forward(const FstGroupedForwardArgs& a, cudaStream_t st) {
  if (a.prob.dtype == FST_F32) return forward_t<float>(a, st);
  if (a.prob.dtype == FST_BF16) return forward_t<__nv_bfloat16>(a, st);
  return forward_t<__half>(a, st);
}

int simt_backward(const FstGroupedBackwardArgs& a, cudaStream_t st) {
  if (a.prob.dtype == FST_F32) return backward_t<float>(a, st);
  if (a.prob.dtype == FST_BF16) return backward_t<__nv_bfloat16>(a, st);
  return backward_t<__half>(a, st);
}

}  // namespace grouped
}  // namespace fst
