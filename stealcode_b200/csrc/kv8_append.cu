// kv8_append.cu -- writing new key/value rows into the paged 8-bit cache,
// and reading stored rows back.
//
// A block is `block` consecutive tokens of one (layer, sequence, kv head)
// that share a scale.  Appending rows x to a block with scale s0 (0 when the
// call writes the block's first token: whatever the page held before is
// forgotten) and a = max |x| over the finite new elements:
//   s    = max(s0, a * (1 / 127))     (a < 1e-30 counts as 0)
//   code = clamp(rint(x * (1 / s)), -127, 127), NaN -> 0, and 0 when s = 0
//   the block's older codes, when s > s0:  rint(code * (s0 / s))
// in IEEE f32 with ties to even: the same rows give the same bits whichever
// kernel writes them.  An element that is not finite takes no part in a, so
// it cannot spoil its neighbours' precision; it is stored as +-127 * s.
#include "kv8.cuh"

namespace sc {
namespace kv8 {

constexpr float kTiny = 1e-30f;

__device__ __forceinline__ float finite_mag(float x) {
  const float a = fabsf(x);
  return a <= 3.402823466e38f ? a : 0.0f;  // false for Inf and NaN
}

__device__ __forceinline__ int8_t code_of(float x, float inv) {
  const float r = rintf(__fmul_rn(x, inv));
  if (r != r) return 0;  // NaN, and Inf * 0
  return (int8_t)(int)fminf(fmaxf(r, -127.0f), 127.0f);
}

// One warp writes one touched block of one head, of K (z = 0) or V (z = 1).
template <typename T, int D>
__global__ void __launch_bounds__(128) append_kernel(const AppendArgs p, int blocks_per_seq) {
  const Layer &c = p.c;
  const int lane = threadIdx.x & 31;
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int i = (int)(unit / blocks_per_seq), bi = (int)(unit % blocks_per_seq);
  if (i >= p.b.m || *c.status) return;
  const int s = p.b.seq(i, c.n_seqs);
  if (s < 0) {
    if (lane == 0) atomicOr(c.status, kBadSeq);
    return;
  }
  int64_t row0;
  int count;
  p.b.rows(i, row0, count);
  const int len = seq_length(c, s), first = len - count;
  // rows before position 0 (more new rows than the sequence holds) are left out
  const int lo = first < 0 ? 0 : first;
  const int blk = lo / c.block + bi;  // index of this block in the sequence
  const int b0 = blk * c.block;
  const int from = lo > b0 ? lo : b0, to = len < b0 + c.block ? len : b0 + c.block;
  if (from >= to) return;
  const int pid = c.table[(int64_t)s * c.max_pages + page_of(c, b0)];
  if ((unsigned)pid >= (unsigned)c.n_pages) {
    if (lane == 0) atomicOr(c.status, kBadPage);
    return;
  }
  const int h = blockIdx.y, z = blockIdx.z;
  const T *src = (const T *)(z ? p.v : p.k) + (int64_t)h * (z ? p.v_head : p.k_head);
  const int64_t ld = z ? p.v_row : p.k_row;
  const int slot0 = b0 - page_of(c, b0) * c.page;
  const int64_t ph = (int64_t)pid * c.kv + h;
  int8_t *dst = (z ? c.v : c.k) + (ph * c.page + slot0) * D;
  float *sp = (z ? c.vs : c.ks) + ph * (c.page / c.block) + slot0 / c.block;

  constexpr int E = D / 32;  // elements of a row per lane
  float a = 0.0f;
#pragma unroll 4
  for (int t = from; t < to; t++) {
    const T *r = src + (row0 + t - first) * ld + lane * E;
#pragma unroll
    for (int e = 0; e < E; e++) a = fmaxf(a, finite_mag(to_f32<T>(r[e])));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
  const float s0 = from > b0 ? *sp : 0.0f;
  const float want = a >= kTiny ? __fmul_rn(a, 1.0f / 127.0f) : 0.0f;
  const float sc = fmaxf(s0, want);
  const float inv = sc > 0.0f ? __fdiv_rn(1.0f, sc) : 0.0f;
  if (from > b0 && sc > s0) {
    const float ratio = __fdiv_rn(s0, sc);
    for (int t = b0; t < from; t++) {
      int8_t *d = dst + (t - b0) * D + lane * E;
#pragma unroll
      for (int e = 0; e < E; e++) d[e] = (int8_t)(int)rintf(__fmul_rn((float)d[e], ratio));
    }
  }
#pragma unroll 4
  for (int t = from; t < to; t++) {
    const T *r = src + (row0 + t - first) * ld + lane * E;
    int8_t *d = dst + (t - b0) * D + lane * E;
#pragma unroll
    for (int e = 0; e < E; e++) d[e] = code_of(to_f32<T>(r[e]), inv);
  }
  __syncwarp();
  if (lane == 0) *sp = sc;
}

template <typename T, int D>
static int launch_append(const AppendArgs &a, cudaStream_t st) {
  const int per = (int)ceil_div(a.b.n - 1, a.c.block) + 1;  // blocks n rows can touch
  dim3 grid((unsigned)ceil_div((int64_t)a.b.m * per, 4), a.c.kv, 2);
  append_kernel<T, D><<<grid, 128, 0, st>>>(a, per);
  SC_CUDA(cudaGetLastError());
  note_launch();
  return kOk;
}

int append(const AppendArgs &a, cudaStream_t st) {
  if (a.b.m == 0 || a.b.n == 0) return kOk;
  const bool wide = a.head_dim == 128;
  if (a.dtype == SC_DTYPE_F32)
    return wide ? launch_append<float, 128>(a, st) : launch_append<float, 64>(a, st);
  if (a.dtype == SC_DTYPE_F16)
    return wide ? launch_append<__half, 128>(a, st) : launch_append<__half, 64>(a, st);
  return wide ? launch_append<__nv_bfloat16, 128>(a, st) : launch_append<__nv_bfloat16, 64>(a, st);
}

// ---- reading back --------------------------------------------------------------

// One warp per (row, head): code * scale; tokens without a page read as 0.
template <typename T, int D>
__global__ void __launch_bounds__(128) rows_kernel(const RowsArgs p) {
  const Layer &c = p.c;
  const int lane = threadIdx.x & 31;
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int i = (int)(unit / p.b.n), j = (int)(unit % p.b.n);
  if (i >= p.b.m) return;
  int64_t row0;
  int count;
  p.b.rows(i, row0, count);
  if (j >= count) return;
  const int s = p.b.seq(i, c.n_seqs);
  if (s < 0 && lane == 0) atomicOr(c.status, kBadSeq);
  const int tok = s < 0 ? -1 : seq_length(c, s) - count + j;
  const int pid = tok < 0 ? -1 : c.table[(int64_t)s * c.max_pages + page_of(c, tok)];
  const bool ok = (unsigned)pid < (unsigned)c.n_pages;
  const int h = blockIdx.y, slot = tok < 0 ? 0 : tok - page_of(c, tok) * c.page;
  const int64_t ph = (int64_t)(ok ? pid : 0) * c.kv + h;
  constexpr int E = D / 32;
#pragma unroll
  for (int z = 0; z < 2; z++) {
    T *out = (T *)(z ? p.v : p.k);
    if (!out) continue;
    out += ((row0 + j) * c.kv + h) * D + lane * E;
    float sc = 0.0f;
    if (ok) sc = (z ? c.vs : c.ks)[ph * (c.page / c.block) + slot / c.block];
    const int8_t *src = (z ? c.v : c.k) + (ph * c.page + slot) * D + lane * E;
#pragma unroll
    for (int e = 0; e < E; e++) out[e] = from_f32<T>(ok ? __fmul_rn((float)src[e], sc) : 0.0f);
  }
}

template <typename T, int D>
static int launch_rows(const RowsArgs &a, cudaStream_t st) {
  dim3 grid((unsigned)ceil_div((int64_t)a.b.m * a.b.n, 4), a.c.kv);
  rows_kernel<T, D><<<grid, 128, 0, st>>>(a);
  SC_CUDA(cudaGetLastError());
  note_launch();
  return kOk;
}

int read_rows(const RowsArgs &a, cudaStream_t st) {
  if (a.b.m == 0 || a.b.n == 0 || (!a.k && !a.v)) return kOk;
  const bool wide = a.head_dim == 128;
  if (a.dtype == SC_DTYPE_F32) return wide ? launch_rows<float, 128>(a, st) : launch_rows<float, 64>(a, st);
  if (a.dtype == SC_DTYPE_F16) return wide ? launch_rows<__half, 128>(a, st) : launch_rows<__half, 64>(a, st);
  return wide ? launch_rows<__nv_bfloat16, 128>(a, st) : launch_rows<__nv_bfloat16, 64>(a, st);
}

}  // namespace kv8
}  // namespace sc
