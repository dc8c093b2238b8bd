// kv8_attend_tile.cu -- attention over the paged 8-bit cache for many query
// rows per kv head (prompts, long chunks), on the tensor cores' own memory.
// Formulas and numerics are kv8_attend.cu's, with one reference for a row's sum
// and its output (e = 2^(x - m), w = e * vs * gain * 2^8, m bounds
// x + log2(vs * gain)) and two gains for the value scales; the parts of split
// items and the sharing-out are kv8_work.cuh's.
//
// A block takes 256 rows (token, query head of the group) as two tiles of 128
// and walks the keys 128 at a time:
//   warps 0-7, 8-15 softmax of row tile 0, 1: two threads hold a row, read 64
//                   of its scores each from tensor memory, write the weights
//                   back over them as f16, and rescale the output
//                   accumulator when its maximum has grown by more than 2^7;
//   warps 16-19     read the codes of K and V (16-byte loads, one tile ahead
//                   in registers) and write them to shared memory as f16
//                   operands: K as it lies (its depth is contiguous), V
//                   transposed by stmatrix;
//   warps 20, 21    issue S = Q K^T and O += W V of row tile 0, 1: while one
//                   row tile is in its softmax the other's products run.  A
//                   warp each, since a row tile's chain (softmax, W V, the
//                   next Q K^T over the weights just read) waits for a barrier
//                   at every step and one warp would wait for both in turn;
//   warp 22         runs one piece ahead and sends its queries and first keys
//                   to L2.
// The codes pass through the converters once for 256 rows, so their cost is
// shared by all query heads of the group.
//
// Operands are no-swizzle K-major: element (row, k) of an operand of R rows
// is at ((k / 8) * R + row) * 16 + (k % 8) * 2 bytes.  Within 64 elements of
// V's depth the order is n = 8 p + 2 t + e for element 16 t + 2 p + e: what a
// lane's 16 loaded bytes give stmatrix without a shuffle; the epilogue undoes
// it.  f32 queries and weights are hi + lo pairs of f16: twice the products.
//
// Measured: a prompt of 4096 tokens, 32 heads of 128 on 8, bf16: 247 us, 557
// TFLOP/s of the visible pairs (of 1642 measured for bf16 products); 64 x 750
// f32 frames, 8 heads: 385 us; four chunks of 301-1024 tokens, 16 heads of 64
// on 4, window 2048: 86 us.  Bound by a row tile's chain: softmax 3 k cycles,
// its two products 1.6 k (M 128 from shared memory takes 102 cycles a 16-deep
// step instead of 64), a barrier wake-up after each; the tensor pipe is a
// quarter busy.  Items of few key tiles also pay for queries, result and, where
// they are split, the join (10-20 k cycles).
#include <atomic>

#include "kv8_work.cuh"
#include "sc_kernels.cuh"
#include "sc_tcgen05.cuh"

namespace sc {
namespace kv8 {

constexpr int kTileRows = 256, kTileKeys = 128;
constexpr int kTileThreads = 768;  // 23 warps work; setmaxnreg takes whole warpgroups
// Registers a thread: 80 at launch, which the 16 softmax warps keep; the four
// product warps give 32 each to the converters (16 * 80 + 4 * 112 + 4 * 48 = 24 * 80).
// With 72 for the softmax and 128 for the converters the softmax spills into
// its loop: a prompt of 4096 tokens 274 us, so 247.
constexpr int kTileRegs = 80;
// An item's queries and result cost about as much as three tiles (a prompt of
// 4096 tokens with 2, 3, 5, 8, an earlier version: 271, 254, 259, 273 us).
constexpr int kTileOver = 3;
constexpr float kTileShift = 256.0f, kTileSlack = 7.0f;
constexpr float kTinyFactor = 1e-37f;  // a score factor of 0 would make NaN of a hidden score's -inf

// The value scales vs that a piece computes with are vs * gain, so that a
// row's sum l of 2^(x - m), where m bounds x + log2(vs * gain), stays inside
// f32 with bits to spare.  Gain 2^8: exponents from -80 (vs = 2^72) to 98.6
// (the smallest scale, 1e-30 / 127), to which up to 7 (m's slack) and the
// tokens' number are added.  A piece of work that meets a larger vs goes on
// with gain 2^-40 (up to vs = 2^121, the largest): its old results are scaled
// by 2^-48, and scales below 2^-60 are held against 2^-60 then, so what a row
// draws from them loses bits and at last vanishes beside those of 2^72.
constexpr float kGain = 256.0f, kGainLog2 = 8.0f, kBigGain = 0x1p-40f, kBigScale = 0x1p72f;
constexpr float kToBig = 0x1p-48f, kFromBig = 0x1p48f, kToBigLog2 = -48.0f;
constexpr float kLeastLog2 = -100.0f;  // of vs * gain
constexpr float kBigSum = 0x1p60f;     // sums above it are not scaled by 2^48
constexpr float kPartUnit = 0x1p-8f;   // of a part's output: results from 1e-30 to f32's largest have room

// l * 2^d for a sum l, f = 2^d: with scales far apart 2^d can underflow
// where the product does not.
__device__ __forceinline__ float scale_sum(float l, float d, float f) {
  if (d > -100.0f) return l * f;
  const float h = exp2_approx(0.5f * d);
  return l * h * h;
}

template <int D, bool SPLIT>
struct TileCfg {
  static constexpr int kStages = SPLIT && D == 128 ? 1 : 2;
  static constexpr int kQ = 128 * D * 2;   // bytes of one row tile's queries (one term)
  static constexpr int kKv = 128 * D * 2;  // bytes of one K or V tile
  static constexpr int kTerms = SPLIT ? 2 : 1;
  static constexpr int kOperands = 2 * kTerms * kQ + 2 * kStages * kKv;
};

struct TileShared {  // after the operands
  uint64_t q_full[2], s_full[2], p_full[2], pv_done[2];
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2];
  // a key tile's 16-token groups: score factor ks, log2(vs * gain), weight
  // factor vs * gain * 2^8 (slots 0-3 for kGain, 4-7 for kBigGain), and whether
  // the group has a page (bit 8: the piece has come to a scale above kBigScale,
  // so its gain is kBigGain); four tiles deep, so a slot is written again only
  // after both softmaxes have gone through the next tile too
  float kf[8][8], lv[8][8], wf[8][8];
  uint32_t live[4][4];  // two bits from each converter warp, and bit 8
  float top[2][2][2][128];  // [tile parity][row tile][half][row]: largest score, and once a piece the sums
  float sum[2][2][128];     // [row tile][half][row] sums where the gain turns to kBigGain
  ShareScratch share;
  uint32_t tmem;
  int last;
  volatile int started;  // pieces the softmax warps have begun
};

// Which groups of a tile have a page (bits 0-7), and whether its gain is kBigGain.
__device__ __forceinline__ uint32_t live_word(const TileShared &sh, int slot) {
  return sh.live[slot][0] | sh.live[slot][1] | sh.live[slot][2] | sh.live[slot][3];
}

__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void soft_sync() { asm volatile("bar.sync 1, 512;" ::: "memory"); }

// The eight warps of a row tile.
__device__ __forceinline__ void tile_sync(int q) { asm volatile("bar.sync %0, 256;" ::"r"(10 + q) : "memory"); }
// The two warps that hold the halves of 32 rows.
__device__ __forceinline__ void pair_sync(int id) { asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory"); }

__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void tc_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
      "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
      "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void stmatrix_t(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b),
               "r"(c), "r"(d)
               : "memory");
}

__device__ __forceinline__ void tc_st16(uint32_t taddr, const uint32_t *r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
      : "memory");
}

// The lowest n bits.
__device__ __forceinline__ uint32_t below(int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u; }

// 8 consecutive elements of a result row.
template <typename T>
__device__ __forceinline__ void store_row(T *dst, const float (&v)[8], int vec) {
  if (vec) {
    constexpr int W = 16 / sizeof(T);
#pragma unroll
    for (int e = 0; e < 8; e += W) {
      uint4 w;
      T *x = reinterpret_cast<T *>(&w);
#pragma unroll
      for (int u = 0; u < W; u++) x[u] = from_f32<T>(v[e + u]);
      *(uint4 *)(dst + e) = w;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++) dst[e] = from_f32<T>(v[e]);
  }
}

// 8 rows of q as f16 (hi and, for f32, lo), each scaled by a power of two
// with the sign of the score factor.  Lane = (row of the 8, one of 4 16-byte
// pieces): every load takes 64 contiguous bytes of a row, and every store 8
// consecutive rows of an operand chunk, which share no bank.  src: the lane's
// row, or nullptr (zeros).  Writes the row's score factor to *factor.
template <int D, typename T>
__device__ __forceinline__ void load_queries(const T *src, bool vec, float scale, unsigned char *hi, unsigned char *lo,
                                             float *factor) {
  constexpr int N = 16 / sizeof(T), S = D / (4 * N);  // elements of a piece, 64-byte segments of a row
  const int piece = (threadIdx.x >> 3) & 3;
  uint4 raw[S];
#pragma unroll
  for (int i = 0; i < S; i++) {
    raw[i] = make_uint4(0, 0, 0, 0);
    if (src && vec) raw[i] = __ldg((const uint4 *)src + i * 4 + piece);
  }
  if (src && !vec) {
#pragma unroll
    for (int i = 0; i < S; i++) {
      T *x = reinterpret_cast<T *>(&raw[i]);
#pragma unroll
      for (int e = 0; e < N; e++) x[e] = src[(i * 4 + piece) * N + e];
    }
  }
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < S; i++) {
    const T *x = reinterpret_cast<const T *>(&raw[i]);
#pragma unroll
    for (int e = 0; e < N; e++) top = fmaxf(top, fabsf(to_f32<T>(x[e])));
  }
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
  int k = 0;
  if (top > 0.0f) k = min(100, 140 - (int)(__float_as_uint(top) >> 23));
  float up = __uint_as_float((uint32_t)(127 + k) << 23);
  const float down = __uint_as_float((uint32_t)(127 - k) << 23);
  // score factors stay positive: a group's largest score is its largest product
  if (scale < 0.0f) up = -up;
  if (scale == 0.0f) up = 0.0f;
  if (piece == 0) *factor = fabsf(scale) * kLog2e * down;
#pragma unroll
  for (int i = 0; i < S; i++) {
    const T *x = reinterpret_cast<const T *>(&raw[i]);
    if constexpr (sizeof(T) == 2) {  // 8 elements: a chunk's row
      uint32_t h[4];
#pragma unroll
      for (int e = 0; e < 4; e++) h[e] = pack_f16(to_f32<T>(x[2 * e]) * up, to_f32<T>(x[2 * e + 1]) * up);
      *(uint4 *)(hi + (i * 4 + piece) * 2048) = make_uint4(h[0], h[1], h[2], h[3]);
    } else {  // 4 elements: half of it
      uint32_t h[2], l[2];
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const float a = to_f32<T>(x[2 * e]) * up, b = to_f32<T>(x[2 * e + 1]) * up;
        h[e] = pack_f16(a, b);
        const float2 y = __half22float2(*reinterpret_cast<const __half2 *>(&h[e]));
        l[e] = pack_f16(a - y.x, b - y.y);
      }
      const int at = (i * 2 + (piece >> 1)) * 2048 + (piece & 1) * 8;
      *(uint2 *)(hi + at) = make_uint2(h[0], h[1]);
      *(uint2 *)(lo + at) = make_uint2(l[0], l[1]);
    }
  }
}

template <int D, typename T>
__global__ void __launch_bounds__(kTileThreads, 1)
    attend_tile_kernel(const __grid_constant__ AttendArgs p, const __grid_constant__ WorkGrid g, int vec_q, int vec_o) {
  constexpr bool SPLIT = sizeof(T) == 4;
  using C = TileCfg<D, SPLIT>;
  constexpr int NS = C::kStages;
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned char *qs = smem;                             // [2 row tiles][terms] queries
  unsigned char *kt = smem + 2 * C::kTerms * C::kQ;     // [NS] K tiles
  unsigned char *vt = kt + NS * C::kKv;                 // [NS] V tiles
  TileShared &sh = *reinterpret_cast<TileShared *>(vt + NS * C::kKv);
  const Layer &c = p.c;
  const int tid = (int)threadIdx.x, warp = tid >> 5, lane = tid & 31;

  Share share;
  if (!find_share<kTileRows, kTileKeys, kTileOver, kTileThreads>(p, g, sh.share, share)) return;
  if (tid == 0) {
    sh.started = 0;
    for (int i = 0; i < 2; i++) {
      mbar_init(&sh.q_full[i], 8);
      mbar_init(&sh.s_full[i], 2);  // the MMA thread's own arrival and its commit
      mbar_init(&sh.p_full[i], 8);
      mbar_init(&sh.pv_done[i], 1);
      mbar_init(&sh.k_full[i], 4);
      mbar_init(&sh.k_empty[i], 2);  // both MMA warps
      mbar_init(&sh.v_full[i], 4);
      mbar_init(&sh.v_empty[i], 2);
    }
    fence_barrier_init();
  }
  if (warp == 20) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;  // columns: S0 0, S1 128, O0 256, O1 384
  bool ok = true;
  Entry en;
  Piece pc;

  if (warp < 16) {
    // ================= softmax =================
    const int q = warp >> 3, half = (warp >> 2) & 1, row = (warp & 3) * 32 + lane;
    const int pair = 2 + q * 4 + (warp & 3);  // named barrier of this warp and the one with the rows' other half
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_at = tmem + lanes + (uint32_t)(q * 128 + half * 64), o_at = tmem + lanes + (uint32_t)(256 + q * 128);
    int ns = 0;   // tiles this row tile has gone through
    int nk = 0;   // key tiles of the block (slots of the scale ring)
    // a wait that gave up (ok false) is the last one of its thread; the loops
    // run to their end, so every warp reaches the same barriers
    while (next_piece<kTileRows, kTileKeys, kTileOver>(p, g, share, en, pc)) {
      const int nt = max(0, min(pc.t1, en.tiles()) - pc.t0);
      const int nr = en.r1 - en.r0;
      const bool on = q * 128 < nr;          // this row tile has rows
      const int r = en.r0 + q * 128 + row;   // row of the sequence
      const bool mine = r < en.r1;
      int j, hq;
      en.row(g, q * 128 + row, j, hq);
      hq += pc.head * g.group;
      const int pos = mine ? en.first + j : -1;
      float m = -INFINITY, l = 0.0f;
      bool big = false;  // the gain at the piece's end
      if (tid == 0) sh.started = sh.started + 1;
      if (on && nt > 0) {
        // the pair of warps loads its 32 rows, 16 each
#pragma unroll 1
        for (int i = 0; i < 2; i++) {
          const int lr = (warp & 3) * 32 + half * 16 + i * 8 + (lane & 7), r2 = en.r0 + q * 128 + lr;
          int j2, h2;
          en.row(g, q * 128 + lr, j2, h2);
          unsigned char *hi = qs + q * C::kTerms * C::kQ + lr * 16;
          load_queries<D, T>(
              r2 < en.r1 ? (const T *)p.q + (en.row0 + j2) * p.q_row + (pc.head * g.group + h2) * p.q_head : nullptr,
              vec_q, p.scale, hi, hi + C::kQ, &sh.top[1][q][0][lr]);
        }
        pair_sync(pair);
        const float qf = sh.top[1][q][0][row];
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.q_full[q]);
        // positions of the row tile's first and last row
        int j_lo, j_hi, h_any;
        en.row(g, q * 128, j_lo, h_any);
        en.row(g, min(nr, q * 128 + 128) - 1, j_hi, h_any);
        const int p_lo = en.first + j_lo, p_hi = en.first + j_hi;
        for (int x = 0; x < nt; x++, ns++) {
          if (ok) ok = mbar_wait(&sh.s_full[q], (uint32_t)ns & 1u);
          __syncwarp();
          tc_fence_after();
          const uint32_t live = live_word(sh, (nk + x) & 3);
          const int slot = ((nk + x) & 3) + (int)(live >> 8) * 4;
          if (live > 0xffu) sh.sum[q][half][row] = l;
          const int t0 = en.tile(pc.t0 + x) * kTileKeys;
          const bool all = (live & 0xffu) == 0xffu && t0 + kTileKeys - 1 <= p_lo &&
                           (p.window <= 0 || t0 > p_hi - p.window || t0 + kTileKeys - 1 < p.sinks);
          if (!all) {  // -inf over what the row does not see, in tensor memory
#pragma unroll 1
            for (int i = 0; i < 2; i++) {
              const int c0 = half * 64 + 32 * i, d = pos - t0 - c0 + 1;
              uint32_t see = below(d);
              if (p.window > 0) see &= ~below(d - p.window) | below(p.sinks - t0 - c0);
              const uint32_t lv = live >> (c0 >> 4);
              see &= (lv & 1u ? 0xffffu : 0u) | (lv & 2u ? 0xffff0000u : 0u);
              uint32_t s[32];
              tc_ld<32>(s_at + 32 * i, s);
              tc_wait_ld<32>(s);
#pragma unroll
              for (int e = 0; e < 32; e++)
                if (!((see >> e) & 1u)) s[e] = 0xff800000u;
              tc_st32(s_at + 32 * i, s);
            }
            tc_wait_st();
          }
          // The scores are read twice, 32 columns at a time, in loops: the
          // code of the four roles has to stay inside the instruction cache.
          float top = -INFINITY;
#pragma unroll 1
          for (int i = 0; i < 2; i++) {
            uint32_t s[32];
            tc_ld<32>(s_at + 32 * i, s);
            const int gr = half * 4 + 2 * i;
            const float f0 = fmaxf(sh.kf[slot][gr] * qf, kTinyFactor), f1 = fmaxf(sh.kf[slot][gr + 1] * qf, kTinyFactor);
            const float v0 = sh.lv[slot][gr], v1 = sh.lv[slot][gr + 1];
            tc_wait_ld<32>(s);
            float a = __uint_as_float(s[0]), b = __uint_as_float(s[16]);
#pragma unroll
            for (int e = 1; e < 16; e++) {
              a = fmaxf(a, __uint_as_float(s[e]));
              b = fmaxf(b, __uint_as_float(s[16 + e]));
            }
            top = fmaxf(top, fmaxf(a * f0 + v0, b * f1 + v1));
          }
          sh.top[x & 1][q][half][row] = top;
          pair_sync(pair);
          top = fmaxf(top, sh.top[x & 1][q][half ^ 1][row]);
          bool grow = top > m + (x ? kTileSlack : 0.0f);
          if (__any_sync(0xffffffffu, grow || live > 0xffu)) {
            float f = 1.0f;  // factor of the output accumulator
            if (live > 0xffu && x && live_word(sh, (nk + x - 1) & 3) <= 0xffu) {  // the gain turns
              if (fmaxf(l, sh.sum[q][half ^ 1][row]) <= kBigSum) {  // the same O under a smaller bound
                l *= kFromBig;
                m += kToBigLog2;
              } else {
                f = kToBig;
              }
              grow = top > m + kTileSlack;
            }
            const float now = grow ? top : m;
            const float fl = grow ? exp2_approx(m - now) : 1.0f;
            if (grow) l = scale_sum(l, m - now, fl);
            m = now;
            f *= fl;
            if (x) {  // every product into O before this tile's has completed (see the MMA warp)
#pragma unroll 1
              for (int i = half * (D / 64); i < (half + 1) * (D / 64); i++) {
                uint32_t o[32];
                tc_ld<32>(o_at + 32 * i, o);
                tc_wait_ld<32>(o);
#pragma unroll
                for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                tc_st32(o_at + 32 * i, o);
              }
            }
          }
          const float nm = m == -INFINITY ? 0.0f : -m;
          const uint64_t nm2 = pack2(nm, nm);
          uint64_t l2 = 0;
#pragma unroll 1
          for (int i = 0; i < 2; i++) {
            uint32_t s[32];
            tc_ld<32>(s_at + 32 * i, s);
            const int gr = half * 4 + 2 * i;
            float f[2], wf[2];
#pragma unroll
            for (int h = 0; h < 2; h++) {
              f[h] = fmaxf(sh.kf[slot][gr + h] * qf, kTinyFactor);
              wf[h] = sh.wf[slot][gr + h];
            }
            tc_wait_ld<32>(s);
            // 32 keys: 16 columns of packed weights (and 16 of their low
            // terms) over the scores just read
            uint32_t w[32];
#pragma unroll
            for (int e = 0; e < 16; e++) {
              const int h = e / 8;
              const uint64_t a = ffma2((uint64_t)s[2 * e] | ((uint64_t)s[2 * e + 1] << 32), pack2(f[h], f[h]), nm2);
              const uint64_t b = pack2(exp2_approx(lo_of(a)), exp2_approx(hi_of(a)));
              l2 = fadd2(l2, b);
              const uint64_t v = fmul2(b, pack2(wf[h], wf[h]));
              w[e] = pack_f16(lo_of(v), hi_of(v));
              if (SPLIT) {
                const float2 y = __half22float2(*reinterpret_cast<const __half2 *>(&w[e]));
                w[16 + e] = pack_f16(lo_of(v) - y.x, hi_of(v) - y.y);
              }
            }
            if constexpr (SPLIT) {
              tc_st32(s_at + 32 * i, w);
            } else {
              tc_st16(s_at + 32 * i, w);
            }
          }
          l += lo_of(l2) + hi_of(l2);
          big = live > 0xffu;
          tc_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.p_full[q]);
        }
        // the row's sum from both halves
        sh.top[nt & 1][q][half][row] = l;
        pair_sync(pair);
        l += sh.top[nt & 1][q][half ^ 1][row];
        pair_sync(pair);  // read before the next piece's queries write there
      }
      nk += nt;
      // ---- the piece's result ----
      const int kPart = kTileRows * (D + 2);
      float *part = g.parts + (int64_t)(pc.starts ? 2 * (int)blockIdx.x + 1 : 2 * (int)blockIdx.x) * kPart;
      if (on) {
        if (nt > 0) {
          if (ok) ok = mbar_wait(&sh.pv_done[q], (uint32_t)(ns - 1) & 1u);
          __syncwarp();
          tc_fence_after();
        }
        const int pr = q * 128 + row;  // row of the item
        // A whole item: O / (l * units).  A part: its sum is brought to [1, 2), its
        // output along with it and, whatever the gain was, to units of kPartUnit:
        // parts join under one reference, and nothing leaves f32's range.
        const float units = kTileShift * (big ? kBigGain : kGain);
        float inv = l == 0.0f ? 0.0f : 1.0f / l, unit = 1.0f / units;
        if (!pc.whole && l > 0.0f && l < INFINITY) {
          const uint32_t bits = __float_as_uint(l);
          const int k = (int)(bits >> 23) - 127;
          inv = exp2_approx((float)-k);
          unit *= kPartUnit;
          m += (float)k;
          l = __uint_as_float((bits & 0x7fffffu) | 0x3f800000u);
        }
        T *dst = (T *)p.out + (en.row0 + j) * p.o_row + hq * p.o_head;
        // A whole item's rows go through the queries' shared memory (their
        // last product has completed), 16-byte pieces swizzled by the row, so
        // that both the writes here and the rows' stores below run over whole
        // lines: a thread's own row would be a line for each lane.
        constexpr int RB = D * sizeof(T);  // bytes of a row
        unsigned char *stage = qs + q * C::kTerms * C::kQ;
        const bool staged = pc.whole && vec_o;
        if (staged) tile_sync(q);  // no warp still reads the queries' sums or stages of the piece before
#pragma unroll 1
        for (int i = half * (D / 64); i < (half + 1) * (D / 64); i++) {
          uint32_t o[32];
          if (nt > 0) {
            tc_ld<32>(o_at + 32 * i, o);
            tc_wait_ld<32>(o);
          } else {
#pragma unroll
            for (int e = 0; e < 32; e++) o[e] = 0;
          }
#pragma unroll
          for (int t = 0; t < 4; t++) {  // 8 consecutive elements
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = __uint_as_float(o[8 * (e / 2) + 2 * t + (e & 1)]) * inv * unit;
            const int d0 = (i >> 1) * 64 + t * 16 + (i & 1) * 8;
            if (staged) {
              constexpr int W = 16 / sizeof(T);
#pragma unroll
              for (int e = 0; e < 8; e += W) {
                uint4 w;
                T *x = reinterpret_cast<T *>(&w);
#pragma unroll
                for (int u = 0; u < W; u++) x[u] = from_f32<T>(v[e + u]);
                *(uint4 *)(stage + row * RB + ((((d0 + e) / W) ^ (row & 7)) * 16)) = w;
              }
            } else if (mine) {
              if (!pc.whole) {
                *(float4 *)(part + (int64_t)pr * D + d0) = make_float4(v[0], v[1], v[2], v[3]);
                *(float4 *)(part + (int64_t)pr * D + d0 + 4) = make_float4(v[4], v[5], v[6], v[7]);
              } else {
#pragma unroll
                for (int e = 0; e < 8; e++) dst[d0 + e] = from_f32<T>(v[e]);
              }
            }
          }
        }
        if (staged) {
          pair_sync(pair);
          constexpr int L = RB / 16;  // lanes of a row
#pragma unroll 4
          for (int i = 0; i < 16; i += 32 / L) {
            const int lr = (warp & 3) * 32 + half * 16 + i + lane / L, r2 = en.r0 + q * 128 + lr;
            if (r2 < en.r1) {
              int j2, h2;
              en.row(g, q * 128 + lr, j2, h2);
              const uint4 w = *(const uint4 *)(stage + lr * RB + (((lane % L) ^ (lr & 7)) * 16));
              *(uint4 *)((T *)p.out + (en.row0 + j2) * p.o_row + (pc.head * g.group + h2) * p.o_head +
                         (lane % L) * (16 / sizeof(T))) = w;
            }
          }
          tile_sync(q);  // the next piece's queries may be written
        }
        if (mine && half == 0) {
          if (pc.whole) {
            if (p.lse) p.lse[(en.row0 + j) * p.n_heads + hq] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
          } else {
            part[kTileRows * D + pr] = m;
            part[kTileRows * D + kTileRows + pr] = l;
          }
        }
        tc_fence_before();  // O has been read before the next piece's first product overwrites it
      }
      if (!pc.whole) {
        // the block that finishes the item last joins its parts
        __threadfence();
        soft_sync();
        if (tid == 0) {
          const int done = atomicAdd(&g.count[pc.c0], 1);
          sh.last = done == pc.parts - 1;
          if (sh.last) g.count[pc.c0] = 0;
        }
        soft_sync();
        if (sh.last) {
          __threadfence();
          // a thread joins 8 elements of a row, in one pass: a part's loads
          // wait for nothing before them, four parts are on their way
          for (int u = tid; u < nr * (D / 8); u += 512) {
            const int rr = u / (D / 8), d0 = u % (D / 8) * 8;
            float top = -INFINITY, sum = 0.0f, acc[8];
#pragma unroll
            for (int e = 0; e < 8; e++) acc[e] = 0.0f;
#pragma unroll 4
            for (int k = 0; k < pc.parts; k++) {
              const float *y = g.parts + (int64_t)part_slot(pc.c0, k) * kPart;
              const float pm = __ldcg(y + kTileRows * D + rr), pl = __ldcg(y + kTileRows * D + kTileRows + rr);
              const float4 va = __ldcg((const float4 *)(y + rr * D + d0)), vb = __ldcg((const float4 *)(y + rr * D + d0) + 1);
              const float now = fmaxf(top, pm);
              const float old = now == -INFINITY ? 1.0f : exp2_approx(top - now);
              const float f = pm == -INFINITY ? (pl != pl ? pl : 0.0f) : exp2_approx(pm - now);
              top = now;
              sum = sum * old + f * pl;
              const float v[8] = {va.x, va.y, va.z, va.w, vb.x, vb.y, vb.z, vb.w};
#pragma unroll
              for (int e = 0; e < 8; e++) acc[e] = acc[e] * old + f * v[e];
            }
            int j2, h2;
            en.row(g, rr, j2, h2);
            h2 += pc.head * g.group;
            const float inv = sum == 0.0f ? 0.0f : 1.0f / (sum * kPartUnit);
            T *dst = (T *)p.out + (en.row0 + j2) * p.o_row + h2 * p.o_head + d0;
#pragma unroll
            for (int e = 0; e < 8; e++) acc[e] *= inv;
            store_row<T>(dst, acc, vec_o);
            if (p.lse && d0 == 0)
              p.lse[(en.row0 + j2) * p.n_heads + h2] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * kLn2;
          }
        }
        soft_sync();  // sh.last is free
      }
    }
  } else if (warp < 20) {
    // ================= converters =================
    asm volatile("setmaxnreg.inc.sync.aligned.u32 112;");
    const int w = warp - 16;
    constexpr int HF = D / 64;
    const int nblk = c.page / c.block;
    int nk = 0;
    while (next_piece<kTileRows, kTileKeys, kTileOver>(p, g, share, en, pc)) {
      const int nt = max(0, min(pc.t1, en.tiles()) - pc.t0);
      if (nt == 0) continue;
      const int32_t *trow = c.table + (int64_t)en.s * c.max_pages;
      // this warp's tokens of a tile: groups 2 w and 2 w + 1
      auto pages = [&](int x, int (&pid)[2]) {
#pragma unroll
        for (int u = 0; u < 2; u++) {
          const int tok = en.tile(pc.t0 + x) * kTileKeys + w * 32 + u * 16;
          const bool in = x < nt && tok <= en.p_hi &&
                          (p.window <= 0 || tok + 15 > en.p_lo - p.window || tok < p.sinks);
          const int id = in ? trow[page_of(c, tok)] : -1;
          pid[u] = (unsigned)id < (unsigned)c.n_pages ? id : -1;
          if (id >= c.n_pages && lane == 0) atomicOr(c.status, kBadPage);
        }
      };
      auto base = [&](int x, int u, int pid) {  // the group's first row of codes
        const int tok = en.tile(pc.t0 + x) * kTileKeys + w * 32 + u * 16;
        return ((int64_t)pid * c.kv + pc.head) * c.page + tok - page_of(c, tok) * c.page;
      };
      uint4 kr[4][HF], vr[4][HF];
      float ks = 1.0f, vs = 1.0f;  // lanes 0, 1: the scales of the warp's groups
      uint32_t large = 0;
      auto load_k = [&](int x, const int (&pid)[2]) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int id = pid[i >> 1];
          if (id >= 0) {
            const int8_t *src = c.k + (base(x, i >> 1, id) + (i & 1) * 8 + (lane & 7)) * D + (lane >> 3) * 16;
#pragma unroll
            for (int h = 0; h < HF; h++) kr[i][h] = __ldg((const uint4 *)(src + h * 64));
          } else {
#pragma unroll
            for (int h = 0; h < HF; h++) kr[i][h] = make_uint4(0, 0, 0, 0);
          }
        }
        ks = vs = 1.0f;
        if (lane < 2) {
          const int id = lane ? pid[1] : pid[0];
          if (id >= 0) {
            const int tok = en.tile(pc.t0 + x) * kTileKeys + w * 32 + lane * 16;
            const int slot = tok - page_of(c, tok) * c.page;
            const int64_t at = ((int64_t)id * c.kv + pc.head) * nblk + (slot >> c.block_shift);
            ks = __ldg(c.ks + at);
            vs = __ldg(c.vs + at);
          }
        }
      };
      auto load_v = [&](int x, const int (&pid)[2]) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int id = pid[i >> 1];
          if (id >= 0) {
            const int8_t *src = c.v + (base(x, i >> 1, id) + (i & 1) * 8 + (lane >> 2)) * D + (lane & 3) * 16;
#pragma unroll
            for (int h = 0; h < HF; h++) vr[i][h] = __ldg((const uint4 *)(src + h * 64));
          } else {
#pragma unroll
            for (int h = 0; h < HF; h++) vr[i][h] = make_uint4(0, 0, 0, 0);
          }
        }
      };
      int pid[2], nxt[2];
      pages(0, pid);
      load_k(0, pid);
      load_v(0, pid);
      pages(1, nxt);
      for (int x = 0; x < nt; x++, nk++) {
        const int st = nk % NS;
        const uint32_t turn = (uint32_t)(nk / NS) & 1u;
        if (ok) ok = mbar_wait(&sh.k_empty[st], turn ^ 1u);
        __syncwarp();
        unsigned char *kd = kt + st * C::kKv;
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
          for (int h = 0; h < HF; h++) {
            const uint32_t a[4] = {kr[i][h].x, kr[i][h].y, kr[i][h].z, kr[i][h].w};
            uint32_t o[8];
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const uint32_t y = a[e] ^ 0x80808080u;
              o[2 * e] = two_f16(y, kLow);
              o[2 * e + 1] = two_f16(y, kHigh);
            }
            const int tok = w * 32 + i * 8 + (lane & 7), kc = h * 8 + (lane >> 3) * 2;
            *(uint4 *)(kd + (kc * 128 + tok) * 16) = make_uint4(o[0], o[1], o[2], o[3]);
            *(uint4 *)(kd + ((kc + 1) * 128 + tok) * 16) = make_uint4(o[4], o[5], o[6], o[7]);
          }
        const int slot = nk & 3;
        if (lane < 2) {
          // a scale of 0 has codes of 0: any factor does that keeps the weights inside f16
          const float v = vs > 0.0f ? vs : 1.0f / kGain;
          const float lv = log2_approx(v) + kGainLog2;
          const int gr = 2 * w + lane;
          sh.kf[slot][gr] = sh.kf[slot + 4][gr] = ks > 0.0f ? ks : 1.0f;
          sh.lv[slot][gr] = lv;
          sh.lv[slot + 4][gr] = fmaxf(lv + kToBigLog2, kLeastLog2);
          sh.wf[slot][gr] = v * (kTileShift * kGain);
          sh.wf[slot + 4][gr] = v * (kTileShift * kBigGain);
        }
        if (__any_sync(0xffffffffu, lane < 2 && vs > kBigScale)) large = 0x100u;
        if (lane == 0) sh.live[slot][w] = ((pid[0] >= 0 ? 1u : 0u) | (pid[1] >= 0 ? 2u : 0u)) << (2 * w) | large;
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.k_full[st]);
        if (x + 1 < nt) load_k(x + 1, nxt);
        if (ok) ok = mbar_wait(&sh.v_empty[st], turn ^ 1u);
        __syncwarp();
        const uint32_t vd = smem_u32(vt + st * C::kKv);
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
          for (int h = 0; h < HF; h++) {
            const uint32_t a[4] = {vr[i][h].x, vr[i][h].y, vr[i][h].z, vr[i][h].w};
            uint32_t o[8];
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const uint32_t y = a[e] ^ 0x80808080u;
              o[2 * e] = two_f16(y, kLow);
              o[2 * e + 1] = two_f16(y, kHigh);
            }
            // matrices p = 0..3 then 4..7; lane gives the address of row (lane & 7) of matrix lane / 8
            const uint32_t at = vd + (uint32_t)(((w * 4 + i) * D + h * 64 + (lane >> 3) * 8 + (lane & 7)) * 16);
            stmatrix_t(at, o[0], o[1], o[2], o[3]);
            stmatrix_t(at + 32 * 16, o[4], o[5], o[6], o[7]);
          }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.v_full[st]);
        if (x + 1 < nt) load_v(x + 1, nxt);
        pid[0] = nxt[0];
        pid[1] = nxt[1];
        if (x + 2 < nt) pages(x + 2, nxt);
      }
    }
  } else {
    // ================= MMA =================
    asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
    if (warp < 22) {
      // the whole warp walks the tiles (so that addresses stay in uniform
      // registers) and polls the barriers, one lane issues
      const bool lead = elect_one();
      const int q = __shfl_sync(0xffffffffu, warp - 20, 0);
      const uint32_t id_s = umma_idesc_f16(128), id_o = umma_idesc_f16(D);
      const uint64_t qd = umma_desc(qs + q * C::kTerms * C::kQ, 2048, 128), k0 = umma_desc(kt, 2048, 128),
                     v0 = umma_desc(vt, D * 16, 128);
      const uint32_t s_at = tmem + q * 128, o_at = tmem + 256 + q * 128;
      int np = 0, nq = 0, nk = 0;  // products into O, pieces with this row tile, key tiles
      // S from K stage st, once the last product that read its weights (they
      // lie over the scores) has completed
      auto scores = [&](int x) {
        const int st = (nk + x) % NS;
        if (!mbar_wait(&sh.k_full[st], (uint32_t)((nk + x) / NS) & 1u)) return false;
        if (np > 0 && !mbar_wait(&sh.pv_done[q], (uint32_t)(np - 1) & 1u)) return false;
        tc_fence_after();
        if (lead) {
          const uint64_t kd = k0 + (uint64_t)((st * C::kKv) >> 4);
#pragma unroll
          for (int t = 0; t < C::kTerms; t++)  // low terms first: less of them is lost to the large sums
#pragma unroll
            for (int i = 0; i < D / 16; i++)
              tc_mma_f16(s_at, qd + (uint64_t)(((C::kTerms - 1 - t) * C::kQ + i * 4096) >> 4),
                         kd + (uint64_t)((i * 4096) >> 4), id_s, (uint32_t)(t | i));
          mbar_arrive(&sh.s_full[q]);
          tc_commit(&sh.s_full[q]);
          tc_commit(&sh.k_empty[st]);
        }
        return true;
      };
      auto output = [&](int x) {
        const int st = (nk + x) % NS;
        if (!mbar_wait(&sh.v_full[st], (uint32_t)((nk + x) / NS) & 1u)) return false;
        if (!mbar_wait(&sh.p_full[q], (uint32_t)np & 1u)) return false;
        tc_fence_after();
        if (lead) {
          const uint64_t vd = v0 + (uint64_t)((st * C::kKv) >> 4);
#pragma unroll
          for (int t = 0; t < C::kTerms; t++)
#pragma unroll
            for (int i = 0; i < 8; i++)
              tc_mma_ts(o_at, s_at + (i >> 1) * 32 + t * 16 + (i & 1) * 8, vd + (uint64_t)((i * 2 * D * 16) >> 4), id_o,
                        t | i ? 1u : (uint32_t)x);
          tc_commit(&sh.pv_done[q]);
          tc_commit(&sh.v_empty[st]);
        }
        return true;
      };
      while (ok && next_piece<kTileRows, kTileKeys, kTileOver>(p, g, share, en, pc)) {
        const int nt = max(0, min(pc.t1, en.tiles()) - pc.t0);
        if (nt == 0) continue;
        if (q == 0 || en.r1 - en.r0 > 128) {
          ok = mbar_wait(&sh.q_full[q], (uint32_t)nq++ & 1u) && scores(0);
          for (int x = 0; x < nt && ok; x++) {
            ok = output(x);
            np++;
            if (ok && x + 1 < nt) ok = scores(x + 1);
            ok = __all_sync(0xffffffffu, ok);  // a lane whose wait gave up ends the loop for all
          }
        } else {  // no rows here: the tiles are released unread
          for (int x = 0; x < nt && ok; x++) {
            const int st = (nk + x) % NS;
            const uint32_t turn = (uint32_t)((nk + x) / NS) & 1u;
            ok = mbar_wait(&sh.k_full[st], turn);
            if (ok && lead) mbar_arrive(&sh.k_empty[st]);
            ok = ok && mbar_wait(&sh.v_full[st], turn);
            if (ok && lead) mbar_arrive(&sh.v_empty[st]);
            ok = __all_sync(0xffffffffu, ok);
          }
        }
        ok = __all_sync(0xffffffffu, ok);
        nk += nt;
      }
      // every product completes before the tensor memory is released
      if (np > 0 && !mbar_wait(&sh.pv_done[q], (uint32_t)(np - 1) & 1u)) ok = false;
    }
    if (warp == 22) {
      int n = 0;
      const long long t0 = clock64();
      while (next_piece<kTileRows, kTileKeys, kTileOver>(p, g, share, en, pc)) {
        // one piece ahead of the softmax warps; a hint only, so it gives up quietly
        while (sh.started < n && clock64() - t0 < kWaitCycles) __nanosleep(200);
        n++;
        if (pc.t0 >= en.tiles()) continue;
        if (vec_q)
          for (int r = en.r0 + lane; r < en.r1; r += 32) {
            int j, h;
            en.row(g, r - en.r0, j, h);
            prefetch_l2((const T *)p.q + (en.row0 + j) * p.q_row + (pc.head * g.group + h) * p.q_head, D * sizeof(T));
          }
        const int tok = en.tile(pc.t0) * kTileKeys + (lane >> 1) * 16, pi = page_of(c, tok);
        if (lane < 16 && tok <= en.p_hi) {
          const int pid = c.table[(int64_t)en.s * c.max_pages + pi];
          if ((unsigned)pid < (unsigned)c.n_pages)
            prefetch_l2((lane & 1 ? c.v : c.k) + (((int64_t)pid * c.kv + pc.head) * c.page + tok - pi * c.page) * D, 16 * D);
        }
      }
    }
    __syncwarp();
  }
  if (!ok) atomicOr(c.status, kWaitTimeout);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 20)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

template <int D, typename T>
static int launch_tile(const AttendArgs &a, int sm_count, cudaStream_t st) {
  using C = TileCfg<D, sizeof(T) == 4>;
  WorkGrid g;
  g.group = a.n_heads / a.c.kv;
  g.magic = (uint32_t)((2097152 + g.group - 1) / g.group);
  g.per_seq = (int)ceil_div((int64_t)a.b.n * g.group, kTileRows);
  g.entries = a.b.m * g.per_seq;
  // Where there are fewer units than blocks could take: a share of u tiles of an
  // item of n costs u tiles' time and n / u parts to join, each by its rows, so
  // u near sqrt(n rows / 256) (4 heads of 128, bf16; shares of 2, 4, 8, 16: 256
  // rows over 2048 tokens 53, 48, 55, 79 us, over 8192 121, 83, 72, 86; 64 rows
  // over 8192 42, 35, 38, 53).  Items of a few tiles are not split: 256 rows
  // over 512 tokens 26 us whole, 36 in shares of 2.
  int64_t keys = a.max_len;
  if (a.window > 0 && (int64_t)a.window + a.b.n + a.sinks + 2 * kTileKeys < keys)
    keys = (int64_t)a.window + a.b.n + a.sinks + 2 * kTileKeys;
  const int64_t tiles = ceil_div(keys, kTileKeys), all = (int64_t)a.b.n * g.group, rows = all < kTileRows ? all : kTileRows;
  g.min_share = 2;
  while ((int64_t)g.min_share * g.min_share * kTileRows < tiles * rows && g.min_share < 64) g.min_share++;
  if (tiles + kTileOver <= 8) g.min_share = (int)tiles + kTileOver;
  g.count = (int32_t *)a.ws;
  g.parts = (float *)((char *)a.ws + kMaxBlocks * 4);
  const bool vq = ((uintptr_t)a.q & 15) == 0 && a.q_row * sizeof(T) % 16 == 0 && a.q_head * sizeof(T) % 16 == 0;
  const bool vo = ((uintptr_t)a.out & 15) == 0 && a.o_row * sizeof(T) % 16 == 0 && a.o_head * sizeof(T) % 16 == 0;
  static std::atomic<size_t> limit[64];
  const size_t bytes = C::kOperands + sizeof(TileShared);
  const int rc = raise_smem_limit((const void *)attend_tile_kernel<D, T>, bytes, limit);
  if (rc) return rc;
  // the converters would wait for registers that a smaller launch does not have
  static std::atomic<bool> checked{false};
  if (!checked.load(std::memory_order_relaxed)) {
    cudaFuncAttributes f;
    SC_CUDA(cudaFuncGetAttributes(&f, (const void *)attend_tile_kernel<D, T>));
    if (f.numRegs < kTileRegs) {
      set_error("kv8_attend: built with %d registers a thread, %d are needed", f.numRegs, kTileRegs);
      return kErrUnsupported;
    }
    checked.store(true, std::memory_order_relaxed);
  }
  attend_tile_kernel<D, T><<<sm_count, kTileThreads, bytes, st>>>(a, g, vq, vo);
  SC_CUDA(cudaGetLastError());
  note_launch();
  return kOk;
}

size_t tile_ws_bytes(int sm_count) { return (size_t)sm_count * 2 * kTileRows * 130 * 4; }

int attend_tile(const AttendArgs &a, int sm_count, cudaStream_t st) {
  const bool wide = a.head_dim == 128;
  if (a.dtype == SC_DTYPE_F32) return wide ? launch_tile<128, float>(a, sm_count, st) : launch_tile<64, float>(a, sm_count, st);
  if (a.dtype == SC_DTYPE_F16) return wide ? launch_tile<128, __half>(a, sm_count, st) : launch_tile<64, __half>(a, sm_count, st);
  return wide ? launch_tile<128, __nv_bfloat16>(a, sm_count, st) : launch_tile<64, __nv_bfloat16>(a, sm_count, st);
}

}  // namespace kv8
}  // namespace sc
