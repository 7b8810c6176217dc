// C-ABI entry points of the grouped-head attention and of the rotary
// positions: argument validation and the choice of kernels. Errors come back
// as status codes with a thread-local message; nothing throws or aborts.

#include <cuda_runtime.h>
#include <math.h>

#include <cstdint>
#include <initializer_list>

#include "fst_grouped.cuh"

namespace {

using fst::api_fail;

constexpr int64_t kMaxRows = (1ll << 31) - 256;

int check_grouped(const FstGroupedProblem& p) {
  if (p.dtype < FST_F32 || p.dtype > FST_F16)
    return api_fail(FST_ERR_INVALID, "unknown dtype %d", p.dtype);
  if (p.batch < 0 || p.heads <= 0 || p.kv_heads <= 0 || p.head_dim <= 0 || p.total_rows < 0 ||
      p.max_len < 0)
    return api_fail(FST_ERR_INVALID, "bad sizes B=%d H=%d Hkv=%d Dh=%d", p.batch, p.heads,
                    p.kv_heads, p.head_dim);
  if (p.heads % p.kv_heads)
    return api_fail(FST_ERR_INVALID, "the query heads (%d) must be a multiple of the key heads (%d)",
                    p.heads, p.kv_heads);
  if (p.head_dim > 128)
    return api_fail(FST_ERR_UNSUPPORTED, "Dh (=%d) must be <= 128", p.head_dim);
  if (!isfinite(p.scale)) return api_fail(FST_ERR_INVALID, "scale must be finite");
  if (p.flags) return api_fail(FST_ERR_INVALID, "unknown flags 0x%x", (unsigned)p.flags);
  if (p.packed < 0 || p.packed > 1)
    return api_fail(FST_ERR_INVALID, "unknown layout %d (0 padded, 1 packed)", p.packed);
  if (p.total_rows > kMaxRows)
    return api_fail(FST_ERR_UNSUPPORTED, "%lld rows: at most %lld", (long long)p.total_rows,
                    (long long)kMaxRows);
  if (p.packed) {
    if (!p.cu_seqlens) return api_fail(FST_ERR_INVALID, "packed needs cu_seqlens");
  } else {
    if (!p.seqlens && p.total_rows > 0) return api_fail(FST_ERR_INVALID, "padded needs seqlens");
    if ((int64_t)p.batch * p.max_len != p.total_rows)
      return api_fail(FST_ERR_INVALID, "padded total_rows must equal B*L");
  }
  // One block per 64 rows and head is the finest grid a kernel launches.
  if (fst::grouped::list_blocks(p, 64) * p.heads >= (1ll << 31))
    return api_fail(FST_ERR_UNSUPPORTED, "%lld rows of %d heads are too many",
                    (long long)p.total_rows, p.heads);
  return FST_OK;
}

bool any_null(std::initializer_list<const void*> ptrs) {
  for (const void* p : ptrs)
    if (!p) return true;
  return false;
}

// An address that is not a multiple of its element's size would fault on the GPU.
bool misaligned(size_t size, std::initializer_list<const void*> ptrs) {
  for (const void* p : ptrs)
    if ((uintptr_t)p % size) return true;
  return false;
}
size_t size_of(int dtype) { return dtype == FST_F32 ? 4 : 2; }

int status(const char* where) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return api_fail(FST_ERR_CUDA, "%s: %s", where, cudaGetErrorString(e));
  return FST_OK;
}

int check_rotary(const FstRotaryArgs& p) {
  if (p.dtype < FST_F32 || p.dtype > FST_F16)
    return api_fail(FST_ERR_INVALID, "unknown dtype %d", p.dtype);
  if (p.batch < 0 || p.heads <= 0 || (p.k.data && p.kv_heads <= 0) || p.total_rows < 0 ||
      p.max_len < 0)
    return api_fail(FST_ERR_INVALID, "bad sizes B=%d H=%d Hkv=%d", p.batch, p.heads, p.kv_heads);
  if (p.head_dim < 1 || p.head_dim > 1024)
    return api_fail(FST_ERR_UNSUPPORTED, "Dh (=%d) must be 1 to 1024", p.head_dim);
  if (p.pairs < 0 || 2 * (int64_t)p.pairs > p.head_dim)
    return api_fail(FST_ERR_INVALID, "%d channel pairs do not fit Dh = %d", p.pairs, p.head_dim);
  if (!isfinite(p.magnitude)) return api_fail(FST_ERR_INVALID, "magnitude must be finite");
  if (p.packed < 0 || p.packed > 1)
    return api_fail(FST_ERR_INVALID, "unknown layout %d (0 padded, 1 packed)", p.packed);
  if (!p.packed && (int64_t)p.batch * p.max_len != p.total_rows)
    return api_fail(FST_ERR_INVALID, "padded total_rows must equal B*L");
  if (p.total_rows > 0) {
    if (p.packed && !p.positions && !p.cu_seqlens)
      return api_fail(FST_ERR_INVALID, "packed rows need cu_seqlens or positions");
    if (!p.q.data || !p.q_out.data || (p.k.data && !p.k_out.data) || (p.pairs > 0 && !p.freqs))
      return api_fail(FST_ERR_INVALID, "rotary: a required pointer is null");
    if (misaligned(size_of(p.dtype), {p.q.data, p.k.data, p.q_out.data, p.k_out.data}) ||
        misaligned(8, {p.freqs}) || misaligned(4, {p.cu_seqlens}) ||
        misaligned(p.positions_64 ? 8 : 4, {p.positions}))
      return api_fail(FST_ERR_INVALID, "rotary: a pointer is not aligned to its elements");
  }
  return FST_OK;
}

}  // namespace

extern "C" {

int fst_grouped_forward(const FstGroupedForwardArgs* a, void* stream) {
  if (!a) return api_fail(FST_ERR_INVALID, "null args");
  const int rc = check_grouped(a->prob);
  if (rc) return rc;
  if (a->prob.total_rows == 0) return FST_OK;
  if (any_null({a->q.data, a->k.data, a->v.data, a->out.data, a->lse}))
    return api_fail(FST_ERR_INVALID, "grouped forward: q, k, v, out and lse are required");
  if (misaligned(size_of(a->prob.dtype), {a->q.data, a->k.data, a->v.data, a->out.data,
                                          a->out_low.data}) ||
      misaligned(4, {a->lse, a->prob.seqlens, a->prob.cu_seqlens}))
    return api_fail(FST_ERR_INVALID, "grouped forward: a pointer is not aligned to its elements");
  cudaGetLastError();  // clear a stale error so the check below is ours
  const cudaStream_t st = (cudaStream_t)stream;
  const int done = fst::grouped::tc_takes(*a) ? fst::grouped::tc_forward(*a, st)
                                              : fst::grouped::simt_forward(*a, st);
  return done ? done : status("grouped forward launch");
}

int fst_grouped_backward(const FstGroupedBackwardArgs* a, void* stream) {
  if (!a) return api_fail(FST_ERR_INVALID, "null args");
  const int rc = check_grouped(a->prob);
  if (rc) return rc;
  if (a->prob.total_rows == 0) return FST_OK;
  if (any_null({a->q.data, a->k.data, a->v.data, a->out.data, a->dout.data, a->dq.data,
                a->dk.data, a->dv.data, a->lse, a->stats}))
    return api_fail(FST_ERR_INVALID, "grouped backward: a required pointer is null");
  if (misaligned(size_of(a->prob.dtype),
                 {a->q.data, a->k.data, a->v.data, a->out.data, a->out_low.data, a->dout.data,
                  a->dq.data, a->dk.data, a->dv.data}) ||
      misaligned(4, {a->lse, a->stats, a->prob.seqlens, a->prob.cu_seqlens}))
    return api_fail(FST_ERR_INVALID, "grouped backward: a pointer is not aligned to its elements");
  cudaGetLastError();
  const cudaStream_t st = (cudaStream_t)stream;
  const int done = fst::grouped::tc_takes(*a) ? fst::grouped::tc_backward(*a, st)
                                              : fst::grouped::simt_backward(*a, st);
  return done ? done : status("grouped backward launch");
}

int fst_rotary(const FstRotaryArgs* a, void* stream) {
  if (!a) return api_fail(FST_ERR_INVALID, "null args");
  const int rc = check_rotary(*a);
  if (rc) return rc;
  if (a->total_rows == 0) return FST_OK;
  cudaGetLastError();
  const int done = fst::launch_rotary(*a, (cudaStream_t)stream);
  return done ? done : status("rotary launch");
}

}  // extern "C"
