// kv8.cuh -- shared definitions of the paged 8-bit key/value cache: the
// device view of a cache, the packing of a call's rows, and the launchers
// (kv8_append.cu, kv8_attend.cu, kv8_pages.cu) behind kv8_api.cu.
//
// Layout.  A page holds `page` consecutive tokens of one sequence for every
// layer and key head: codes int8 [layer][page id][kv head][slot][head_dim],
// so one head's part of a page is contiguous (page * head_dim bytes), and
// one f32 scale per `block` tokens [layer][page id][kv head][page / block].
// A stored value is code * scale.  `page` and `block` are multiples of 16:
// 16 consecutive tokens always share a page and a scale.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/stealcode_b200.h"
#include "sc_common.cuh"

namespace sc {
namespace kv8 {

// Bits of the cache's sticky status word (SC_KV8_* in the header).
enum : unsigned {
  kFullPool = SC_KV8_POOL_FULL,
  kFullTable = SC_KV8_TABLE_FULL,
  kBadSeq = SC_KV8_BAD_SEQUENCE,
  kBadPage = SC_KV8_BAD_PAGE,
  kWaitTimeout = SC_KV8_WAIT_TIMEOUT,
  kBadRows = SC_KV8_BAD_ROWS,
};

// One layer of a cache (pointers already at that layer).
struct Layer {
  int8_t *k, *v;
  float *ks, *vs;
  const int32_t *table;
  const int32_t *length;
  uint32_t *status;
  int n_pages, n_seqs, max_pages;
  int kv, page, block;
  int block_shift;      // log2(block)
  uint32_t page_magic;  // 2^32 / (page / 16), rounded up; 0 for a page of 16
};

// The rows of a call: row r of sequence i (of m) is packed row start(i) + r
// and stands for token length - count(i) + r of sequence seq(i).
struct Batch {
  const int32_t *seqs;  // or nullptr: i
  const int32_t *cu;    // [m + 1], or nullptr: n rows each
  int m, n;
  int64_t total;

  // False for an entry that cu describes wrongly (from a row before the first,
  // to one past the total, fewer than 0 rows or more than n): it has no rows
  // then, so no value of cu leads outside the packed tensors, and none makes
  // some of an entry's rows stand for other tokens.
  __device__ __forceinline__ bool rows(int i, int64_t &start, int &count) const {
    if (!cu) {
      start = (int64_t)i * n;
      count = n;
      return true;
    }
    const int64_t a = cu[i], b = cu[i + 1];
    const bool ok = a >= 0 && b >= a && b <= total && b - a <= n;
    start = ok ? a : 0;
    count = ok ? (int)(b - a) : 0;
    return ok;
  }
  // The sequence of entry i, or -1 (outside the cache).
  __device__ __forceinline__ int seq(int i, int n_seqs) const {
    const int s = seqs ? seqs[i] : i;
    return (unsigned)s < (unsigned)n_seqs ? s : -1;
  }
};

// Length of a sequence, never more than its table row can address.
__device__ __forceinline__ int seq_length(const Layer &c, int s) {
  const int64_t most = (int64_t)c.max_pages * c.page;
  const int n = c.length[s];
  return n < 0 ? 0 : (int64_t)n > most ? (int)most : n;
}

// Page index of a token: n / d with n = token / 16 < 2^26 and d = page / 16
// <= 64 by a product with 2^32 / d rounded up, which is off by less than
// n / 2^32 < 1 / 64: exact, as n / d has no fraction above 1 - 1 / d.
__device__ __forceinline__ int page_of(const Layer &c, int tok) {
  const uint32_t n = (uint32_t)tok >> 4;
  return c.page_magic ? (int)__umulhi(n, c.page_magic) : (int)n;
}

// Starts moving bytes (a multiple of 16, 16-byte aligned) to the L2 cache.
__device__ __forceinline__ void prefetch_l2(const void *p, uint32_t bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(bytes) : "memory");
}

template <typename T>
__device__ __forceinline__ float to_f32(T x);
template <>
__device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// ---- launchers ---------------------------------------------------------------

struct AppendArgs {
  Layer c;
  Batch b;
  const void *k, *v;
  int64_t k_row, k_head, v_row, v_head;  // strides in elements
  int dtype, head_dim;
};
int append(const AppendArgs &a, cudaStream_t st);

struct RowsArgs {
  Layer c;
  Batch b;
  void *k, *v;  // [total][kv][head_dim], either may be null
  int dtype, head_dim;
};
int read_rows(const RowsArgs &a, cudaStream_t st);

struct AttendArgs {
  Layer c;
  Batch b;
  const void *q;
  void *out;
  float *lse;  // [total][n_heads] or nullptr
  int64_t q_row, q_head, o_row, o_head;
  int dtype, head_dim, n_heads;
  float scale;
  int window, sinks;  // window 0: none
  int64_t max_len;    // no sequence is longer (a hint for the launch)
  void *ws;
};
// Bytes of workspace an attend call needs; the part that holds counters has
// to be zero before the first call and is zero again after each call.
size_t attend_ws_bytes(int sm_count);
int attend(const AttendArgs &a, int sm_count, cudaStream_t st);
// kv8_attend_tile.cu: the same for many rows per kv head
size_t tile_ws_bytes(int sm_count);
int attend_tile(const AttendArgs &a, int sm_count, cudaStream_t st);

struct PageArgs {
  int8_t *k, *v;
  float *ks, *vs;
  int32_t *table, *length, *refs;
  uint32_t *status;
  int64_t n_layers;
  int n_pages, n_seqs, max_pages, kv, head_dim, page, block;
  void *ws;
};
size_t page_ws_bytes(int64_t n_pages, int64_t n_seqs, int64_t max_pages);
int reserve(const PageArgs &a, const int32_t *seqs, const int32_t *counts, int m, cudaStream_t st);
int fork(const PageArgs &a, const int32_t *parents, const int32_t *children, int m, int sm_count, cudaStream_t st);
int release(const PageArgs &a, const int32_t *seqs, int m, cudaStream_t st);
int slide(const PageArgs &a, const int32_t *seqs, int m, int window, int sinks, cudaStream_t st);
int compact(const PageArgs &a, int sm_count, cudaStream_t st);

}  // namespace kv8
}  // namespace sc
