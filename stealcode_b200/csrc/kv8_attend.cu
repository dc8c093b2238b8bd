// kv8_attend.cu -- attention over the paged 8-bit cache for few query rows
// per kv head (single tokens, small chunks); kv8_work.cuh says how a call's
// work is shared out.
//
// A row (position p, query head) sees the keys t <= p of its sequence whose
// page it still holds and, with a window w, those with t > p - w or t < sinks.
//   o = sum_t softmax_t(scale * q.k_t) v_t,  lse = log sum_t exp(scale * q.k_t)
// with k_t = code * ks[block of t], and v_t likewise; a row that sees nothing
// gets o = 0, lse = -inf.
//
// Numerics.  The codes are whole numbers and exact in f16.  A row of q is
// scaled by a power of two to a largest magnitude in [2^13, 2^14) and held in
// f16, or as hi + lo in two f16 for f32 inputs (22 bits): an element of a f16
// or bf16 row is exact where it is above 2^-27 (f16) or 2^-30 (bf16: 8 bits) of
// the row's largest, and no element of any type is off by more than 2^-38 of
// that (an f16's smallest step, 2^-24, halved).  Products and sums are f32.  With x = scale * log2(e) * q.k:
//   e = 2^(x - r),  w = e * 2^(log2(vs) + c),  l += e,  O += w * code(v)
// where r bounds x up to 2^64 and r - c + 8 bounds x + log2(vs) up to 2^7: l
// has its own reference, so neither it nor w (f16, or hi + lo of two f16 for
// f32) leaves its range whatever the value scales are.  r and c change when a
// score passes one of the bounds, so the accumulators are rarely rescaled;
// they are whole numbers, so their factors are powers of two.
//
// What bounds it: the codes' bytes, 2 * head_dim a token and kv head.  A warp
// takes 16 tokens at a time with 16-byte loads straight into registers, and
// multiplies codes by queries as S^T = K Q^T (mma.sync m16n8k16, 8 query rows
// to a tile, so few rows waste little): both products contract over an axis
// whose order is free, so K's and V's lanes take the 16 consecutive bytes
// that they load, and nothing passes through shared memory.  The next step's
// codes are sent to L2 meanwhile (64 streams: a seventh more without).
//
// Measured as whole calls, one after the other (GPUs of one kind differ: the
// first case takes 130 to 139 us): 64 sequences of 512-16384 tokens, 32 query
// heads on 8, bf16: 138 us, 4.4 TB/s of codes (of 6.5 measured for a copy); 4
// of 65-131 k tokens: 167 us, 4.7 TB/s.  What is left is instructions: about
// 495 a warp and 16 tokens, of them 160 to turn codes into f16, at 59 % of the
// issue slots; the ALU pipe is at 51 %.  Short pasts are latency (entry, page,
// codes, join: 2-3 us an item): 256 x 7 rows over a window of 560, f32, take
// 88 us for 210 MB.
#include <atomic>

#include "kv8_work.cuh"
#include "sc_kernels.cuh"

namespace sc {
namespace kv8 {

constexpr int kStepTile = 64;    // tokens per tile: 16 for each warp
constexpr int kStepThreads = 128;
constexpr int kStepOver = 1;
constexpr float kShift = 8.0f;     // a row's largest weight is 2^7 .. 2^8 when the references are set,
constexpr float kWide = 15.0f;     // and below 2^15 as long as they are kept
constexpr float kWideSum = 64.0f;  // log2 of a term of l, likewise
constexpr float kNothing = -1e30f; // r of a row that has seen nothing

__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

template <int D, int NT>
struct StepShared {
  static constexpr int kRows = 8 * NT;
  static constexpr int kLd = D + 2;
  uint2 q[2][NT][D / 16][32];       // hi and lo fragments of q
  float qf[kRows];                  // score factor of each row
  float r[4][kRows], u[4][kRows], l[4][kRows];  // of each warp; u = c - r: O is in units of 2^u
  float o[4][kRows][kLd];
  ShareScratch share;
  int last;
};

// The 16 tokens of a warp in one tile.
struct Group {
  int tok;      // first token
  bool live;    // some row sees some of them, and they have a page
  int64_t at;   // offset of the first token's codes, from the head's first
  int64_t sat;  // of its scale
};

template <int D, int NT, typename T>
__global__ void __launch_bounds__(kStepThreads, NT == 1 ? 4 : 3)
    attend_step_kernel(const __grid_constant__ AttendArgs p, const __grid_constant__ WorkGrid g) {
  constexpr int ROWS = 8 * NT;
  constexpr bool kSplit = sizeof(T) == 4;
  constexpr int KS = D / 16;   // k steps of Q.K, and 16-wide d tiles of V
  constexpr int HF = D / 64;   // 64-byte halves of a row
  using S = StepShared<D, NT>;
  extern __shared__ __align__(16) unsigned char smem[];
  S &sh = *reinterpret_cast<S *>(smem);
  const Layer &c = p.c;
  const int tid = (int)threadIdx.x, lane = tid & 31, gi = lane >> 2, ti = lane & 3;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // the same in all lanes: addresses stay in uniform registers

  Share share;
  if (!find_share<ROWS, kStepTile, kStepOver, kStepThreads>(p, g, sh.share, share)) return;
  Entry en;
  Piece pc;
  const int nblk = c.page / c.block;
  const int page_bytes = c.kv * c.page * D, page_scales = c.kv * nblk;  // of one page, K or V
  while (next_piece<ROWS, kStepTile, kStepOver>(p, g, share, en, pc)) {
    const int nr = en.r1 - en.r0;
    // ---- the keys' and values' first loads ----
    const int t1 = min(pc.t1, en.tiles());
    const int32_t *trow = c.table + (int64_t)max(en.s, 0) * c.max_pages;
    const int8_t *kh = c.k + (int64_t)pc.head * c.page * D, *vh = c.v + (int64_t)pc.head * c.page * D;
    const float *ksh = c.ks + pc.head * nblk, *vsh = c.vs + pc.head * nblk;
    auto token = [&](int x) { return x < t1 ? en.tile(x) * kStepTile + warp * 16 : -1; };
    auto page_id = [&](int tok) {
      const bool in = tok >= 0 && tok <= en.p_hi &&
                      (p.window <= 0 || tok + 15 > en.p_lo - p.window || tok < p.sinks);
      return in ? trow[page_of(c, tok)] : -1;
    };
    auto group = [&](int tok, int pid) {
      Group q;
      q.tok = tok;
      q.live = (unsigned)pid < (unsigned)c.n_pages;
      if (!q.live && pid >= 0 && lane == 0) atomicOr(c.status, kBadPage);
      const int slot = tok - page_of(c, tok) * c.page;
      q.at = (int64_t)pid * page_bytes + slot * D;
      q.sat = (int64_t)pid * page_scales + (slot >> c.block_shift);
      return q;
    };
    uint4 kr[2][HF];
    uint32_t vr[4][D / 32];
    float ks = 0.0f, vs = 0.0f;
    auto load_k = [&](const Group &q) {
      if (!q.live) return;
      const int8_t *src = kh + q.at + (gi * D + ti * 16);
#pragma unroll
      for (int u = 0; u < 2; u++)
#pragma unroll
        for (int f = 0; f < HF; f++) kr[u][f] = __ldg((const uint4 *)(src + 8 * u * D + f * 64));
      ks = __ldg(ksh + q.sat);
      vs = __ldg(vsh + q.sat);
    };
    auto load_v = [&](const Group &q) {
      if (!q.live) return;
      const int8_t *base = vh + q.at + (2 * ti * D + gi * (D / 8));
#pragma unroll
      for (int u = 0; u < 4; u++) {
        const int8_t *src = base + ((u & 1) + (u >> 1) * 8) * D;
        if constexpr (D == 128) {
          const uint4 x = __ldg((const uint4 *)src);
          vr[u][0] = x.x; vr[u][1] = x.y; vr[u][2] = x.z; vr[u][3] = x.w;
        } else {
          const uint2 x = __ldg((const uint2 *)src);
          vr[u][0] = x.x; vr[u][1] = x.y;
        }
      }
    };
    // A group's codes are on their way to L2 one step before its loads into
    // registers: HBM's latency is longer than one step of a warp hides.
    auto ahead = [&](const Group &q) {
      if (q.live && lane < 2) prefetch_l2((lane ? vh : kh) + q.at, 16 * D);
    };
    int tok2 = token(pc.t0 + 1);
    Group cur = group(token(pc.t0), page_id(token(pc.t0)));
    int pid2 = page_id(tok2);
    load_k(cur);
    load_v(cur);
    Group nxt = group(tok2, pid2);
    ahead(nxt);
    tok2 = token(pc.t0 + 2);
    pid2 = page_id(tok2);
    // ---- the rows of q: one warp a row ----
    float qv[ROWS / 4][D / 32];
#pragma unroll
    for (int i = 0; i < ROWS / 4; i++) {
      const int r = warp + 4 * i;
      int j, h;
      en.row(g, r, j, h);
      const T *src = (const T *)p.q + (en.row0 + j) * p.q_row + (pc.head * g.group + h) * p.q_head;
#pragma unroll
      for (int e = 0; e < D / 32; e++) qv[i][e] = r < nr ? to_f32<T>(src[e * 32 + lane]) : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < ROWS / 4; i++) {
      const int r = warp + 4 * i;
      float top = 0.0f;
#pragma unroll
      for (int e = 0; e < D / 32; e++) top = fmaxf(top, fabsf(qv[i][e]));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      // 2^k with top * 2^k in [2^13, 2^14); k in [-115, 100] keeps both 2^k and 2^-k normal
      int k = 0;
      if (top > 0.0f) k = min(100, 140 - (int)(__float_as_uint(top) >> 23));
      const float up = __uint_as_float((uint32_t)(127 + k) << 23), down = __uint_as_float((uint32_t)(127 - k) << 23);
      if (lane == 0) sh.qf[r] = p.scale * kLog2e * down;
      __half *hi = (__half *)&sh.q[0][r >> 3][0][0], *lo = (__half *)&sh.q[1][r >> 3][0][0];
#pragma unroll
      for (int e = 0; e < D / 32; e++) {
        const int d = e * 32 + lane;
        // K step and lane whose registers hold element d of a key
        const int at = (((d >> 6) * 4 + ((d & 15) >> 2)) * 32 + (r & 7) * 4 + ((d & 63) >> 4)) * 4 + (d & 3);
        const float x = qv[i][e] * up;
        const __half h = __float2half_rn(x);
        hi[at] = h;
        if (kSplit) lo[at] = __float2half_rn(x - __half2float(h));
      }
    }
    __syncthreads();
    int pos[NT][2];
    float qf[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int u = 0; u < 2; u++) {
        const int r = n * 8 + 2 * ti + u;
        int j, h;
        en.row(g, r, j, h);
        pos[n][u] = r < nr ? en.first + j : -1;
        qf[n][u] = sh.qf[r];
      }

    float o[KS][NT][4];
    float ref[NT][2], off[NT][2], l[NT][2];  // r, c, l
#pragma unroll
    for (int n = 0; n < NT; n++) {
#pragma unroll
      for (int i = 0; i < KS; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) o[i][n][e] = 0.0f;
      ref[n][0] = ref[n][1] = kNothing;
      off[n][0] = off[n][1] = kShift;
      l[n][0] = l[n][1] = 0.0f;
    }

    for (int x = pc.t0; x < t1; x++) {
      const Group nxt2 = group(tok2, pid2);
      ahead(nxt2);
      tok2 = token(x + 3);
      pid2 = page_id(tok2);
      if (!cur.live) {
        load_k(nxt);
        load_v(nxt);
        cur = nxt;
        nxt = nxt2;
        continue;
      }
      // ---- S^T = K Q^T ----
      // four sums for one tile of rows (two for two): a product waits for the
      // one before it in its sum
      constexpr int CH = 4 / NT;
      float s[NT][4], sp[NT][CH][4];
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int u = 0; u < CH; u++)
#pragma unroll
          for (int e = 0; e < 4; e++) sp[n][u][e] = 0.0f;
#pragma unroll
      for (int f = 0; f < HF; f++) {
        const uint32_t w0[4] = {kr[0][f].x, kr[0][f].y, kr[0][f].z, kr[0][f].w};
        const uint32_t w1[4] = {kr[1][f].x, kr[1][f].y, kr[1][f].z, kr[1][f].w};
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const uint32_t x0 = w0[j] ^ 0x80808080u, x1 = w1[j] ^ 0x80808080u;
          const uint32_t a0 = two_f16(x0, kLow), a1 = two_f16(x1, kLow), a2 = two_f16(x0, kHigh),
                         a3 = two_f16(x1, kHigh);
#pragma unroll
          for (int n = 0; n < NT; n++) {
            const uint2 b = sh.q[0][n][f * 4 + j][lane];
            if (kSplit) {
              const uint2 bl = sh.q[1][n][f * 4 + j][lane];
              mma_16816(sp[n][j % (CH / 2)], a0, a1, a2, a3, b.x, b.y);
              mma_16816(sp[n][CH / 2 + j % (CH / 2)], a0, a1, a2, a3, bl.x, bl.y);
            } else {
              mma_16816(sp[n][j % CH], a0, a1, a2, a3, b.x, b.y);
            }
          }
        }
      }
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          s[n][e] = sp[n][0][e] + sp[n][1][e];
          if (CH == 4) s[n][e] += sp[n][CH - 2][e] + sp[n][CH - 1][e];
        }
      const float kf = ks, vf = vs > 0.0f ? vs : 1.0f;
      load_k(nxt);
      // ---- weights ----
      const float lv = log2_approx(vf);
      const bool all = cur.tok + 15 <= en.p_lo &&
                       (p.window <= 0 || cur.tok > en.p_hi - p.window || cur.tok + 15 < p.sinks);
      float most[NT][2];  // no score above these: the references stand
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int u = 0; u < 2; u++) most[n][u] = ref[n][u] + fminf(kWideSum, kWide - (off[n][u] + lv));
      bool grow = false;
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          float v = s[n][e] * (kf * qf[n][e & 1]);
          if (!all) {
            const int tok = cur.tok + gi + (e >> 1) * 8, ps = pos[n][e & 1];
            const bool see = tok <= ps && (p.window <= 0 || tok > ps - p.window || tok < p.sinks);
            v = see ? v : -INFINITY;
          }
          s[n][e] = v;
          grow |= v > most[n][e & 1];
        }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int u = 0; u < 2; u++) {
            float top = fmaxf(s[n][u], s[n][u + 2]);
#pragma unroll
            for (int q = 4; q < 32; q <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, q));
            const float r0 = ref[n][u], r1 = fmaxf(r0, ceilf(top));
            const float b0 = r0 - off[n][u], b1 = fmaxf(b0, ceilf(top + lv) - kShift);  // -u
            const float f = exp2_approx(b0 - b1);
            ref[n][u] = r1;
            off[n][u] = r1 - b1;
            l[n][u] *= exp2_approx(r0 - r1);
#pragma unroll
            for (int i = 0; i < KS; i++) {
              o[i][n][u] *= f;
              o[i][n][u + 2] *= f;
            }
          }
      }
      uint32_t bh[NT][2], bl[NT][2];
#pragma unroll
      for (int n = 0; n < NT; n++) {
        float w[4], wf[2];
#pragma unroll
        for (int u = 0; u < 2; u++) wf[u] = exp2_approx(fminf(off[n][u] + lv, 126.0f));
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const float v = exp2_approx(s[n][e] - ref[n][e & 1]);
          l[n][e & 1] += v;
          w[e] = v * wf[e & 1];
        }
#pragma unroll
        for (int u = 0; u < 2; u++) {
          const uint32_t h = pack_f16(w[2 * u], w[2 * u + 1]);
          bh[n][u] = transpose_8x8(h);
          if (kSplit) {
            const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&h));
            bl[n][u] = transpose_8x8(pack_f16(w[2 * u] - b.x, w[2 * u + 1] - b.y));
          }
        }
      }
      // ---- O^T += V^T W^T ----
#pragma unroll
      for (int wd = 0; wd < D / 32; wd++) {
        const uint32_t x0 = vr[0][wd] ^ 0x80808080u, x1 = vr[1][wd] ^ 0x80808080u;
        const uint32_t x2 = vr[2][wd] ^ 0x80808080u, x3 = vr[3][wd] ^ 0x80808080u;
#pragma unroll
        for (int hf = 0; hf < 2; hf++) {
          const uint32_t e = __byte_perm(x0, x1, hf ? 0x7362 : 0x5140), f = __byte_perm(x2, x3, hf ? 0x7362 : 0x5140);
          const uint32_t a0 = two_f16(e, kLow), a1 = two_f16(e, kHigh), a2 = two_f16(f, kLow), a3 = two_f16(f, kHigh);
#pragma unroll
          for (int n = 0; n < NT; n++) {
            mma_16816(o[wd * 2 + hf][n], a0, a1, a2, a3, bh[n][0], bh[n][1]);
            if (kSplit) mma_16816(o[wd * 2 + hf][n], a0, a1, a2, a3, bl[n][0], bl[n][1]);
          }
        }
      }
      load_v(nxt);
      cur = nxt;
      nxt = nxt2;
    }

    // ---- join the four warps ----
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int u = 0; u < 2; u++) {
        float v = l[n][u];
#pragma unroll
        for (int q = 4; q < 32; q <<= 1) v += __shfl_xor_sync(0xffffffffu, v, q);
        const int r = n * 8 + 2 * ti + u;
        if (gi == 0) {
          sh.r[warp][r] = ref[n][u];
          sh.u[warp][r] = off[n][u] - ref[n][u];
          sh.l[warp][r] = v;
        }
#pragma unroll
        for (int i = 0; i < KS; i++)
          *(float2 *)&sh.o[warp][r][gi * (D / 8) + 2 * i] = make_float2(o[i][n][u], o[i][n][u + 2]);
      }
    __syncthreads();
    const int slot = pc.starts ? 2 * (int)blockIdx.x + 1 : 2 * (int)blockIdx.x;
    constexpr int kPart = ROWS * (D + 3);
    float *part = g.parts + (int64_t)slot * kPart;
    // a warp takes a row, a lane D / 32 of its elements
    constexpr int E = D / 32;
    auto store = [&](int r, float top, float unit, float sum, const float (&acc)[E]) {
      int j, hq;
      en.row(g, r, j, hq);
      hq += pc.head * g.group;
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum, back = exp2_approx(-(top + unit));
      T *dst = (T *)p.out + (en.row0 + j) * p.o_row + hq * p.o_head;
#pragma unroll
      for (int e = 0; e < E; e++) dst[e * 32 + lane] = from_f32<T>(acc[e] * inv * back);
      if (p.lse && lane == 0)
        p.lse[(en.row0 + j) * p.n_heads + hq] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * kLn2;
    };
#pragma unroll
    for (int i = 0; i < ROWS / 4; i++) {
      const int r = warp + 4 * i;
      if (r >= nr) break;
      float top = kNothing, unit = -kNothing, sum = 0.0f, acc[E];
#pragma unroll
      for (int w = 0; w < 4; w++) {
        top = fmaxf(top, sh.r[w][r]);
        unit = fminf(unit, sh.u[w][r]);
      }
#pragma unroll
      for (int e = 0; e < E; e++) acc[e] = 0.0f;
#pragma unroll
      for (int w = 0; w < 4; w++) {
        const float f = exp2_approx(unit - sh.u[w][r]);
        sum += exp2_approx(sh.r[w][r] - top) * sh.l[w][r];
#pragma unroll
        for (int e = 0; e < E; e++) acc[e] += f * sh.o[w][r][e * 32 + lane];
      }
      if (pc.whole) {
        store(r, top, unit, sum, acc);
      } else {
#pragma unroll
        for (int e = 0; e < E; e++) part[r * D + e * 32 + lane] = acc[e];
        if (lane == 0) {
          part[ROWS * D + r] = top;
          part[ROWS * D + ROWS + r] = sum;
          part[ROWS * D + 2 * ROWS + r] = unit;
        }
      }
    }
    if (!pc.whole) {
      __threadfence();
      __syncthreads();
      if (tid == 0) {
        const int done = atomicAdd(&g.count[pc.c0], 1);
        sh.last = done == pc.parts - 1;
        if (sh.last) g.count[pc.c0] = 0;  // ready for the next call
      }
      __syncthreads();
      if (sh.last) {
        __threadfence();
        for (int r = warp; r < nr; r += 4) {
          float top = kNothing, unit = -kNothing;
          for (int k = lane; k < pc.parts; k += 32) {
            const float *q = g.parts + (int64_t)part_slot(pc.c0, k) * kPart + ROWS * D + r;
            top = fmaxf(top, __ldcg(q));
            unit = fminf(unit, __ldcg(q + 2 * ROWS));
          }
#pragma unroll
          for (int q = 16; q > 0; q >>= 1) {
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, q));
            unit = fminf(unit, __shfl_xor_sync(0xffffffffu, unit, q));
          }
          float sum = 0.0f, acc[E];
#pragma unroll
          for (int e = 0; e < E; e++) acc[e] = 0.0f;
#pragma unroll 4
          for (int k = 0; k < pc.parts; k++) {
            const float *q = g.parts + (int64_t)part_slot(pc.c0, k) * kPart;
            const float pr = __ldcg(q + ROWS * D + r), pl = __ldcg(q + ROWS * D + ROWS + r);
            const float f = exp2_approx(unit - __ldcg(q + ROWS * D + 2 * ROWS + r));
            sum += exp2_approx(pr - top) * pl;
#pragma unroll
            for (int e = 0; e < E; e++) acc[e] += f * __ldcg(q + r * D + e * 32 + lane);
          }
          store(r, top, unit, sum, acc);
        }
      }
    }
    __syncthreads();  // shared memory is free for the next piece
  }
}

size_t attend_ws_bytes(int sm_count) {
  const size_t step = (size_t)sm_count * 4 * 2 * 16 * 131 * 4;
  const size_t tile = tile_ws_bytes(sm_count);
  return kMaxBlocks * 4 + (step > tile ? step : tile);
}

template <int D, int NT, typename T>
static int launch_step(const AttendArgs &a, int sm_count, cudaStream_t st) {
  constexpr int ROWS = 8 * NT;
  WorkGrid g;
  g.group = a.n_heads / a.c.kv;
  g.magic = (uint32_t)((2097152 + g.group - 1) / g.group);
  g.per_seq = (int)ceil_div((int64_t)a.b.n * g.group, ROWS);
  g.entries = a.b.m * g.per_seq;
  // A share of u tiles takes about 0.6 us a tile, joining a past of n tiles
  // cut into n / u parts about 0.1 us a part: u near sqrt(n / 6) (a past of
  // 16000 tokens: 24.5 us with shares of 2, 21.6 with 9; 2000 tokens: 11.3
  // and 19.0).
  g.min_share = 2;
  while ((int64_t)g.min_share * g.min_share * 6 * kStepTile < a.max_len && g.min_share < 64) g.min_share++;
  g.count = (int32_t *)a.ws;
  g.parts = (float *)((char *)a.ws + kMaxBlocks * 4);
  // no more blocks than shares there can be
  int64_t keys = a.max_len;
  if (a.window > 0 && (int64_t)a.window + a.b.n + a.sinks + 2 * kStepTile < keys)
    keys = (int64_t)a.window + a.b.n + a.sinks + 2 * kStepTile;
  const int64_t most = ceil_div((ceil_div(keys, kStepTile) + 1 + kStepOver) * g.entries * a.c.kv, g.min_share);
  int64_t blocks = (int64_t)sm_count * (NT == 1 ? 4 : 3);
  if (most < blocks) blocks = most;
  if (blocks < 1) blocks = 1;
  static std::atomic<size_t> limit[64];
  constexpr size_t bytes = sizeof(StepShared<D, NT>);
  const int rc = raise_smem_limit((const void *)attend_step_kernel<D, NT, T>, bytes, limit);
  if (rc) return rc;
  attend_step_kernel<D, NT, T><<<(unsigned)blocks, kStepThreads, bytes, st>>>(a, g);
  SC_CUDA(cudaGetLastError());
  note_launch();
  return kOk;
}

template <typename T>
static int step(const AttendArgs &a, int sm_count, cudaStream_t st) {
  // One tile of 8 rows where a sequence has no more, else two: half as many
  // blocks fit an SM, but 16 rows read the codes once (8 sequences of 4000
  // tokens, 8 rows: 29 us; 16: 36; 24, codes read twice: 49).
  const bool one = (int64_t)a.b.n * (a.n_heads / a.c.kv) <= 8;
  if (a.head_dim == 128) return one ? launch_step<128, 1, T>(a, sm_count, st) : launch_step<128, 2, T>(a, sm_count, st);
  return one ? launch_step<64, 1, T>(a, sm_count, st) : launch_step<64, 2, T>(a, sm_count, st);
}

int attend(const AttendArgs &a, int sm_count, cudaStream_t st) {
  if (a.b.m == 0 || a.b.n == 0 || a.b.total == 0) return kOk;
  // Above 32 rows per kv head the tensor-memory kernel.  8 sequences of 4000
  // tokens, 8 kv heads, 32 rows, here and there: bf16 heads of 128 50 and 56 us,
  // of 64 41 and 45, f32 61 and 73, 43 and 57; 48 rows: 66 and 58, 51 and 45, 80
  // and 74, 55 and 57.  Of 500 tokens: 32 rows 23 and 23 (bf16), 25 and 27 (f32).
  if ((int64_t)a.b.n * (a.n_heads / a.c.kv) > 32) return attend_tile(a, sm_count, st);
  if (a.dtype == SC_DTYPE_F32) return step<float>(a, sm_count, st);
  if (a.dtype == SC_DTYPE_F16) return step<__half>(a, sm_count, st);
  return step<__nv_bfloat16>(a, sm_count, st);
}

}  // namespace kv8
}  // namespace sc
