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
//
// Bound by the rows' bytes, and for few rows by the chain of loads (length,
// page, rows).  12386 f32 rows of 8 heads of 128: 34 us for 127 MB (3.7 TB/s;
// the two-pass kernel below took 81 us, K and V's heads as the slowest grid
// index 40 us); one bf16 row of each of 64 sequences: 3.2 us.
#include "kv8.cuh"

namespace sc {
namespace kv8 {

constexpr float kTiny = 1e-30f;
// Up to this many rows a sequence, a warp takes a block.  A warp and a block of
// threads, 64 sequences, 8 heads of 128, f32: 4 rows 6.8 and 9.5 us, 8 rows 8.3
// and 10.3, 12 rows 10.3 and 10.3, 64 rows 23 and 18.8; 4 sequences: 8 rows 8.3
// and 7, 64 rows 16.5 and 7.  (256 sequences gain from warps up to 32 rows: 27
// and 41.)
constexpr int kStepRows = 8;

__device__ __forceinline__ float finite_mag(float x) {
  const float a = fabsf(x);
  return a <= 3.402823466e38f ? a : 0.0f;  // false for Inf and NaN
}

__device__ __forceinline__ int8_t code_of(float x, float inv) {
  const float r = rintf(__fmul_rn(x, inv));
  if (r != r) return 0;  // NaN, and Inf * 0
  return (int8_t)(int)fminf(fmaxf(r, -127.0f), 127.0f);
}

// One touched block of one head, of K (z = 0) or V (z = 1).
template <typename T>
struct Touched {
  const T *src;      // the row of position `from`
  int64_t ld;        // elements between rows
  int s, h, z;
  int b0, from, to;  // positions: the block's first, new rows [from, to)
  int8_t *dst;       // codes of position b0
  float *scale;
};

// The bi-th block that entry i's rows touch; false if there is none.  Its
// rows can be loaded then; find_page says where they go.  (The status word
// and the page table are read behind the rows: each would be a round trip to
// memory before the first of them.)
template <typename T>
__device__ __forceinline__ bool find_rows(const AppendArgs &p, int i, int bi, int h, int z, bool tell, Touched<T> &o) {
  const Layer &c = p.c;
  if (i >= p.b.m) return false;
  o.s = p.b.seq(i, c.n_seqs);
  if (o.s < 0) {
    if (tell) atomicOr(c.status, kBadSeq);
    return false;
  }
  int64_t row0;
  int count;
  if (!p.b.rows(i, row0, count)) {
    if (tell) atomicOr(c.status, kBadRows);
    return false;
  }
  const int len = seq_length(c, o.s), first = len - count;
  // rows before position 0 (more new rows than the sequence holds) are left out
  const int lo = first < 0 ? 0 : first;
  o.b0 = ((lo >> c.block_shift) + bi) << c.block_shift;
  o.from = max(lo, o.b0);
  o.to = min(len, o.b0 + c.block);
  if (o.from >= o.to) return false;
  o.h = h;
  o.z = z;
  o.ld = z ? p.v_row : p.k_row;
  o.src = (const T *)(z ? p.v : p.k) + h * (z ? p.v_head : p.k_head) + (row0 + o.from - first) * o.ld;
  return true;
}

template <typename T, int D>
__device__ __forceinline__ bool find_page(const Layer &c, bool tell, Touched<T> &o) {
  const int pi = page_of(c, o.b0), pid = c.table[(int64_t)o.s * c.max_pages + pi];
  if (*c.status) return false;
  if ((unsigned)pid >= (unsigned)c.n_pages) {
    if (tell) atomicOr(c.status, kBadPage);
    return false;
  }
  const int slot0 = o.b0 - pi * c.page;
  const int64_t ph = (int64_t)pid * c.kv + o.h;
  o.dst = (o.z ? c.v : c.k) + (ph * c.page + slot0) * D;
  o.scale = (o.z ? c.vs : c.ks) + ph * (c.page >> c.block_shift) + (slot0 >> c.block_shift);
  return true;
}

// Many rows: one block of 128 threads holds the new rows of one touched block
// in registers (64 rows of 128 f32 are 64 registers a thread), so they are
// read once, with every load in flight at the same time.
//
// Uneven rows (cu): entry i's touched blocks take the slots from
// cu[i] / block + 2 i, which leaves room for one more block at either end, so
// the grid has total / block + 2 m slots instead of m times the longest
// entry's; a block of threads finds its entry with one load a thread.
template <typename T, int D>
__global__ void __launch_bounds__(128) append_block_kernel(const AppendArgs p, int blocks_per_seq, int vec) {
  constexpr int N = 16 / sizeof(T);  // elements of a load
  constexpr int C = D / N;           // loads of a row
  constexpr int R = 128 / C;         // rows of one pass
  constexpr int P = 64 / R;          // passes over a block of 64
  __shared__ float tops[4];
  __shared__ int found[2];
  const int tid = threadIdx.x, col = tid % C, row = tid / C;
  // the heads of K and V are the fastest index: neighbours read one row's parts
  const int slot = (int)(blockIdx.x / (2u * p.c.kv)), hz = (int)(blockIdx.x - slot * (2u * p.c.kv));
  const int z = hz >= p.c.kv, h = z ? hz - p.c.kv : hz;
  int entry = slot / blocks_per_seq, nth = slot % blocks_per_seq;
  if (p.b.cu) {
    const int sh = p.c.block_shift;
    if (tid == 0) found[0] = -1;
    __syncthreads();
    for (int i = tid; i < p.b.m; i += 128) {
      const int a = (p.b.cu[i] >> sh) + 2 * i, b = (p.b.cu[i + 1] >> sh) + 2 * (i + 1);
      if (slot >= a && slot < b) {
        found[0] = i;
        found[1] = slot - a;
      }
    }
    if (blockIdx.x == 0) {  // one block sees every entry, also those that take no slot
      int64_t row0;
      int count;
      for (int i = tid; i < p.b.m; i += 128)
        if (!p.b.rows(i, row0, count)) atomicOr(p.c.status, kBadRows);
    }
    __syncthreads();
    entry = found[0];
    nth = found[1];
    if (entry < 0) return;
  }
  Touched<T> o;
  if (!find_rows<T>(p, entry, nth, h, z, tid == 0, o)) return;
  const int n = o.to - o.from;
  uint4 w[P];
#pragma unroll
  for (int i = 0; i < P; i++) {
    const int r = row + i * R;
    w[i] = make_uint4(0, 0, 0, 0);
    if (r < n) {
      const T *src = o.src + r * o.ld + col * N;
      if (vec) {
        w[i] = __ldg((const uint4 *)src);
      } else {
        T *x = reinterpret_cast<T *>(&w[i]);
#pragma unroll
        for (int e = 0; e < N; e++) x[e] = src[e];
      }
    }
  }
  if (!__syncthreads_and(find_page<T, D>(p.c, tid == 0, o))) return;
  const float s0 = o.from > o.b0 ? *o.scale : 0.0f;
  float a = 0.0f;
#pragma unroll
  for (int i = 0; i < P; i++) {
    const T *x = reinterpret_cast<const T *>(&w[i]);
#pragma unroll
    for (int e = 0; e < N; e++) a = fmaxf(a, finite_mag(to_f32<T>(x[e])));
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, d));
  if ((tid & 31) == 0) tops[tid >> 5] = a;
  __syncthreads();
  a = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  const float sc = fmaxf(s0, a >= kTiny ? __fmul_rn(a, 1.0f / 127.0f) : 0.0f);
  const float inv = sc > 0.0f ? __fdiv_rn(1.0f, sc) : 0.0f;
  if (s0 < sc && o.from > o.b0) {  // the block's older rows
    const float ratio = __fdiv_rn(s0, sc);
    for (int x = tid; x < (o.from - o.b0) * (D / 4); x += 128) {
      char4 q = ((char4 *)o.dst)[x];
      q.x = (signed char)(int)rintf(__fmul_rn((float)q.x, ratio));
      q.y = (signed char)(int)rintf(__fmul_rn((float)q.y, ratio));
      q.z = (signed char)(int)rintf(__fmul_rn((float)q.z, ratio));
      q.w = (signed char)(int)rintf(__fmul_rn((float)q.w, ratio));
      ((char4 *)o.dst)[x] = q;
    }
  }
  int8_t *dst = o.dst + (o.from - o.b0) * D + col * N;
#pragma unroll
  for (int i = 0; i < P; i++) {
    const int r = row + i * R;
    if (r >= n) continue;
    const T *x = reinterpret_cast<const T *>(&w[i]);
    uint32_t q[N / 4];
#pragma unroll
    for (int e = 0; e < N; e += 4)
      q[e / 4] = (uint32_t)(uint8_t)code_of(to_f32<T>(x[e]), inv) |
                 (uint32_t)(uint8_t)code_of(to_f32<T>(x[e + 1]), inv) << 8 |
                 (uint32_t)(uint8_t)code_of(to_f32<T>(x[e + 2]), inv) << 16 |
                 (uint32_t)(uint8_t)code_of(to_f32<T>(x[e + 3]), inv) << 24;
    if constexpr (N == 4) {
      *(uint32_t *)(dst + r * D) = q[0];
    } else {
      *(uint2 *)(dst + r * D) = make_uint2(q[0], q[1]);
    }
  }
  if (tid == 0) *o.scale = sc;  // every thread read s0 before the barrier
}

// Few rows (a step of single tokens, a small chunk): one warp per block, so
// that 64 sequences of 8 heads are 1024 warps and not 1024 blocks; the rows
// are read twice, the second time from L1.
template <typename T, int D>
__global__ void __launch_bounds__(128) append_kernel(const AppendArgs p, int blocks_per_seq) {
  const int lane = threadIdx.x & 31;
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  Touched<T> o;
  if (!find_rows<T>(p, (int)(unit / blocks_per_seq), (int)(unit % blocks_per_seq), blockIdx.y, blockIdx.z, lane == 0, o))
    return;
  const int b0 = o.b0, from = o.from, to = o.to;

  constexpr int E = D / 32;  // elements of a row per lane
  float a = 0.0f;
#pragma unroll 4
  for (int t = from; t < to; t++) {
    const T *r = o.src + (t - from) * o.ld + lane * E;
#pragma unroll
    for (int e = 0; e < E; e++) a = fmaxf(a, finite_mag(to_f32<T>(r[e])));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
  if (!__all_sync(0xffffffffu, find_page<T, D>(p.c, lane == 0, o))) return;
  int8_t *dst = o.dst;
  float *sp = o.scale;
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
    const T *r = o.src + (t - from) * o.ld + lane * E;
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
  if (a.b.n > kStepRows) {
    auto fits = [](const void *p, int64_t row, int64_t head) {
      return ((uintptr_t)p | (uintptr_t)(row * (int64_t)sizeof(T)) | (uintptr_t)(head * (int64_t)sizeof(T))) % 16 == 0;
    };
    const int vec = fits(a.k, a.k_row, a.k_head) && fits(a.v, a.v_row, a.v_head);
    const int64_t slots = a.b.cu ? (a.b.total >> a.c.block_shift) + 2 * a.b.m + 1 : (int64_t)a.b.m * per;
    if (slots * 2 * a.c.kv > INT32_MAX) {
      set_error("kv8_append: too many rows");
      return kErrInvalid;
    }
    append_block_kernel<T, D><<<(unsigned)(slots * 2 * a.c.kv), 128, 0, st>>>(a, per, vec);
  } else {
    dim3 grid((unsigned)ceil_div((int64_t)a.b.m * per, 4), a.c.kv, 2);
    append_kernel<T, D><<<grid, 128, 0, st>>>(a, per);
  }
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

// One warp per packed row, all its heads (their loads are independent):
// code * scale; tokens without a page read as 0.  With cu the lanes look for
// the row's entry.  12386 rows of 8 heads of 128 as f32: 37 us for 127 MB,
// four fifths of them written (a warp per row and head took 80 us).
template <typename T, int D>
__global__ void __launch_bounds__(128) rows_kernel(const RowsArgs p) {
  const Layer &c = p.c;
  const int lane = threadIdx.x & 31;
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (unit >= p.b.total) return;
  int i = -1;
  if (p.b.cu) {
    for (int e = lane; e < p.b.m; e += 32)
      if (unit >= p.b.cu[e] && unit < p.b.cu[e + 1]) i = e;
    i = __reduce_max_sync(0xffffffffu, i);
    if (unit == 0) {  // one warp sees every entry, also those that hold no row
      int64_t start;
      int count;
      for (int e = lane; e < p.b.m; e += 32)
        if (!p.b.rows(e, start, count)) atomicOr(c.status, kBadRows);
    }
  } else {
    i = (int)((uint32_t)unit / (uint32_t)p.b.n);
  }
  if (i < 0) return;
  int64_t row0;
  int count;
  p.b.rows(i, row0, count);
  const int j = (int)(unit - row0);
  if (j < 0 || j >= count) return;
  const int s = p.b.seq(i, c.n_seqs);
  if (s < 0 && lane == 0) atomicOr(c.status, kBadSeq);
  const int tok = s < 0 ? -1 : seq_length(c, s) - count + j;
  const int pi = tok < 0 ? 0 : page_of(c, tok);
  const int pid = tok < 0 ? -1 : c.table[(int64_t)s * c.max_pages + pi];
  const bool ok = (unsigned)pid < (unsigned)c.n_pages;
  const int slot = ok ? tok - pi * c.page : 0, nblk = c.page >> c.block_shift;
  const int64_t ph = (int64_t)(ok ? pid : 0) * c.kv;
  constexpr int E = D / 32;  // elements of a head per lane
  struct alignas(E) Codes { int8_t q[E]; };
  struct alignas(E * sizeof(T)) Values { T v[E]; };
#pragma unroll 8
  for (int h = 0; h < c.kv; h++) {
#pragma unroll
    for (int z = 0; z < 2; z++) {
      T *out = (T *)(z ? p.v : p.k);
      if (!out) continue;
      Values v;
      Codes x;
      float sc = 0.0f;
      if (ok) {
        sc = __ldg((z ? c.vs : c.ks) + (ph + h) * nblk + (slot >> c.block_shift));
        x = *(const Codes *)((z ? c.v : c.k) + ((ph + h) * c.page + slot) * D + lane * E);
      }
#pragma unroll
      for (int e = 0; e < E; e++) v.v[e] = from_f32<T>(ok ? __fmul_rn((float)x.q[e], sc) : 0.0f);
      *(Values *)(out + ((row0 + j) * c.kv + h) * D + lane * E) = v;
    }
  }
}

template <typename T, int D>
static int launch_rows(const RowsArgs &a, cudaStream_t st) {
  rows_kernel<T, D><<<(unsigned)ceil_div(a.b.total, 4), 128, 0, st>>>(a);
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
