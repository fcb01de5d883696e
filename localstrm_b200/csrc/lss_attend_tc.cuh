// lss_attend_tc.cuh — the attention of lss_attend.cuh for prompt chunks: many query rows per key head,
// on the fifth-generation tensor cores (tcgen05, sums in tensor memory).
#pragma once

#include <type_traits>

#include "lss_attend.cuh"
#include "lss_int4_tc.cuh"

namespace lss {

constexpr int PA_ROWS = 256;   // query rows of a group: two tiles of 128
constexpr int PA_KT = 128;     // tokens of a unit of work
constexpr int PA_HT = 64;      // tokens of a step: of the copies, the widening, the products and the softmax
// Warpgroups: two of a thread per query row, one that widens keys, one that widens values, one with two warps that issue
// products and two that issue copies.  Registers go from the last three to the first two: 8 x 144 + 12 x 64 of 20 x 96.
constexpr int PA_NT = 5 * 128;
constexpr int PA_OP = 2;       // stages of widened keys, and of values: a multiple of the streams
constexpr int PA_EXTRA = 6;    // see pa_extra
constexpr int PA_SC = 16;      // stages of scales: more than the steps between the copies and the softmax
// Stages of keys and values as they come: 64 KB.
__host__ __device__ constexpr int pa_raw(int D) { return D == 64 ? 8 : 4; }
__host__ __device__ constexpr int pa_smem(int D) { return 1024 + 2 * 128 * D * 2 + 2 * PA_OP * PA_HT * D * 2 + pa_raw(D) * 2 * PA_HT * D; }

// D (+)= A B, both operands in shared memory.
__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, bool add) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 a, b;\n mov.b64 a, {%1, %2};\n mov.b64 b, {%3, %4};\n setp.ne.b32 p, %6, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %5, p;\n}\n" ::"r"(d),
      "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"((uint32_t)add)
      : "memory");
}
__device__ __forceinline__ void tc_st8(uint32_t at, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

// Tiles of tokens that the last query of a group sees.
__device__ __forceinline__ int pa_tiles(const AttendArgs& a, const AtRow& w, int mt) {
  const int last = min((mt + 1) * PA_ROWS, w.n * a.per) - 1;
  return (w.len - w.n + last / a.per + 1 + PA_KT - 1) / PA_KT;
}
// Units of work that a group's start and end count for: its queries and results take the time of some tiles (a tile of
// a group of up to 128 rows takes about half as long).  Without them the CTA that got the shortest rows was the last
// one by far (48 rows of 8 to 32 tokens over 50 to 8,000: 353 us, over 4,000 each 239).
__device__ __forceinline__ int pa_extra(const AttendArgs& a, const AtRow& w, int mt) { return w.n * a.per - mt * PA_ROWS <= 128 ? PA_EXTRA : PA_EXTRA / 2; }
static __device__ __forceinline__ int64_t pa_units(const AttendArgs& a, int r) {
  const AtRow w = at_row<PA_ROWS / 8>(a, r);
  int64_t n = 0;
  for (int mt = 0; mt < w.mt; ++mt) n += pa_tiles(a, w, mt) + pa_extra(a, w, mt);
  return n * a.heads;
}
__device__ __forceinline__ int64_t pa_sum(int64_t v, int64_t* scr) {
  v = warp_allreduce(v, [](int64_t p, int64_t q) { return p + q; });
  if ((threadIdx.x & 31) == 0) scr[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int i = 0; i < PA_NT / 32; ++i) v += scr[i];
  return v;
}
// Floats of one piece in the workspace: m, l, W of its rows, the sums, the first positions with NaN.
__host__ __device__ constexpr int pa_piece(int D) { return PA_ROWS * (3 + D) + D; }

// Where 16 bytes (8 values) `q` of row `r` lie in an operand of ROWS rows: panels of 64 columns, a
// 128-byte line per row, pieces permuted by the row (the 128-byte swizzle).
template <int ROWS = 128>
__device__ __forceinline__ uint32_t pa_place(int r, int q) {
  return (uint32_t)((q >> 3) * (ROWS * 128) + r * 128 + (((q & 7) ^ (r & 7)) << 4));
}

// o = softmax(c q K^T) V for groups of 256 query rows (`per` heads times new tokens of one row and key head).
//
// Two streams of work, each a warpgroup with a thread per query row, a warp that issues its products and its own part
// of tensor memory: scores S = Q K^T of 64 tokens (two places of 128 x 64, f32), which the weights replace as f16, and the
// sums O, which stay there for the whole group.  A group of more than 128 rows has a tile of 128 in each stream; in
// one of fewer rows the streams take the same rows and every other step of 64 tokens each, and are added up at the end
// (128 rows over 192,000 tokens and 8 heads: the second warpgroup idle 424 us).
// Keys and values come as e4m3 through bulk copies that one warp issues, 64 KB on their way, and are widened to f16 by four
// warps each into two stages, once for all rows (exact; 16 rows at a time, the widening is what bounds
// lss_attend_kernel here).
// Scales and the power of two of a query row act as in lss_attend_kernel; the weight of V is
// p 2^(m + log2(v scale) - W + 10) from the softmax's own p, one exponential per score.  Both running
// maxima may lag by 2^5, so that O is rarely rescaled.
// NaN among values that all rows of the group see takes its way through the products.  In steps that some rows do not
// see whole it is kept out of them (0 NaN of a masked place would spoil the row) and held as the first position
// per column from which it is seen.
// The units (group, tile of 128 tokens that it sees) are cut into equal ranges, one per CTA; pieces of a
// group are added up by lss_attend_tc_join_kernel.
// Measured (8 key heads of 128): four chunks of 296 to 416 tokens of 32 heads behind 1,000 to 6,000 others 192 us (one warp issuing for both
// streams, codes widened from registers: 222 to 240), D = 64 160; three trees of 64 tokens of 64 heads over 60,000 to 100,000
// 605 to 680 us (0.82 to 0.92 PFLOP/s; the upper end one after the other, when the power cap takes the clock down); 48 trees of 8 to 32 tokens of 32 heads
// over 50 to 8,000 206 to 219 us (the upper end alone with cold caches).  A step of a stream takes about 2,200 cycles: the exponentials of both streams 1,088 (16 per cycle and SM), products 615 a
// stream (48 cycles for 128 x 64 x 16 from shared memory, 64 for 128 x 128 x 16 with the weights in tensor memory), the rest is
// the way of scores and weights through tensor memory and barriers.  A quarter of the exponentials as polynomials:
// 3 % less, groups of 128 rows 1 % more; scores fetched before the weights of the step before are stored: 5 % more.
//
// With TREE (see lss_attend_kernel) a step that holds new tokens begins with a thread's 64 comparisons, kept as
// bits.  NaN among the new tokens' values, which only their own branches see, is looked for again by the rows that see
// them, once a group, where there was any.
//
// The warps go through the groups on their own, held together by the barriers of what they pass on alone: copies and
// widening run ahead into the next group while the softmax finishes one and fetches its queries.  A stage of widened
// keys or values belongs to steps of one parity, so that a stream that takes every other step sees all of its phases.
// A wait knows a phase by its parity, so nobody may be two phases behind a barrier or miss one:
//   qready[q]  a phase per wide group, waited on in every one by the stream's products alone;
//   nready     a phase per narrow group: both softmax warpgroups arrive (the second one's word that it has left the group before: where
//              it has no step, its products would end this group at once, and ofull[1] be two phases on) and the products
//              of both and the second softmax wait, in every one;
//   ofull[q]   a phase per group, seen by the stream's own softmax in every one, and by the second softmax for stream 0 behind nready,
//              so that at most the last phase is under way.
struct PaGroup {  // a group of query rows, and the tiles of it that a CTA takes
  int row, head, mt, tile0, tile1, nt;
  int start, ctx, n, rows, see_last, see_all, i0, i1;  // steps [i0, i1)
  bool narrow, whole;
};
template <bool TREE>
struct PaWalk {
  int64_t base, end;              // first unit of the group (its extra ones come before its tiles), end of the CTA's range
  int row, head, mt, tile0;
  uint32_t steps, groups, wides;  // of earlier groups: their numbers choose stages and phases
  __device__ __forceinline__ bool get(const AttendArgs& a, PaGroup& g) const {
    if (base >= end) return false;
    const AtRow w = at_row<PA_ROWS / 8>(a, row);
    const int64_t upto = end - base - pa_extra(a, w, mt);  // tiles of the group before the end of the range
    g.nt = pa_tiles(a, w, mt);
    g.tile0 = tile0;
    g.tile1 = (int)min((int64_t)g.nt, upto);
    if (upto <= tile0) return false;
    g.row = row;
    g.head = head;
    g.mt = mt;
    g.n = w.n;
    g.start = a.starts[row];
    g.ctx = w.len - w.n;
    g.rows = min(PA_ROWS, w.n * a.per - mt * PA_ROWS);
    g.narrow = g.rows <= 128;
    g.see_last = g.ctx + (mt * PA_ROWS + g.rows - 1) / a.per + 1;
    g.see_all = TREE ? g.ctx : g.ctx + mt * PA_ROWS / a.per + 1;  // tokens that every row of the group sees
    g.whole = tile0 == 0 && g.tile1 == g.nt;
    g.i0 = tile0 * 2;
    g.i1 = min(g.tile1 * 2, (g.see_last + PA_HT - 1) / PA_HT);
    return true;
  }
  __device__ __forceinline__ void next(const AttendArgs& a, const PaGroup& g) {
    steps += g.i1 - g.i0;
    ++groups;
    wides += !g.narrow;
    base += g.nt + (g.narrow ? PA_EXTRA : PA_EXTRA / 2);
    tile0 = 0;
    if (base < end && --mt < 0) {  // next group of the head, next head, next row with work
      if (++head == a.heads) {
        head = 0;
        do ++row; while (row < a.B - 1 && at_row<PA_ROWS / 8>(a, row).n == 0);
      }
      mt = at_row<PA_ROWS / 8>(a, row).mt - 1;
    }
  }
};

template <int D, int DT, bool TREE>
__global__ void __launch_bounds__(PA_NT, 1) lss_attend_tc_kernel(AttendArgs a) {
  constexpr int CH = D / 8;                // 16-byte pieces of a row in f16
  constexpr int OPB = 128 * D * 2;         // bytes of a 128-row operand
  constexpr int STB = PA_HT * D * 2;       // bytes of a step's keys or values, widened
  constexpr int RAWB = PA_HT * D;          // and as they come
  constexpr int RS = pa_raw(D), OP = PA_OP;
  constexpr int PIECES = RAWB / 16 / 128;  // 16-byte pieces of a step's keys (or values) per widening thread
  constexpr uint32_t NOWHERE = 0x7fffffff;
  constexpr int NN = 4;                    // the widening is two steps, so two groups at most, ahead of the softmax
  static_assert(OP % 2 == 0, "a stage belongs to one stream");
  extern __shared__ __align__(1024) unsigned char pa_dyn[];
  __shared__ __align__(8) uint64_t rfull[2][RS], rempty[2][RS], kfull[OP], kempty[OP], vfull[OP], vempty[OP], sfull[2][2], pready[2][2], pvdone[2], ofull[2], qready[2], nready;
  __shared__ uint32_t tmem_base;
  __shared__ int failed;
  __shared__ __align__(16) float2 sscale[PA_SC][4];  // scales of the step's 16-token parts: of K (< 0: not seen), log2 of that of V
  __shared__ uint32_t parts[PA_SC];        // bit p: part p of the step's values is there
  __shared__ int nan_from[NN][D];          // first position with a NaN among the values of a column
  __shared__ int any_nan[NN], branch_nan[NN];  // branch_nan: NaN among the values of new tokens (TREE)
  __shared__ float row_factor[128], state[3][128];
  __shared__ int64_t scr[PA_NT / 32], found_lo;
  __shared__ int found;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  unsigned char* base = pa_dyn + ((1024 - (saddr(pa_dyn) & 1023)) & 1023);
  unsigned char* qs = base;                // two query operands
  unsigned char* ksm = base + 2 * OPB;     // stages of keys
  unsigned char* vsm = ksm + OP * STB;     // stages of values
  unsigned char* raw = vsm + OP * STB;     // stages of both as they come

  if (warp == 0) tc_alloc(&tmem_base, 512);
  if (tid == 0) {
    failed = 0;
    for (int i = 0; i < RS; ++i) {
      for (int h = 0; h < 2; ++h) {
        mbar_init(&rfull[h][i], 1);
        mbar_init(&rempty[h][i], 4);
      }
    }
    for (int i = 0; i < OP; ++i) {
      mbar_init(&kfull[i], 4);
      mbar_init(&vfull[i], 4);
      mbar_init(&kempty[i], 2);
      mbar_init(&vempty[i], 2);
    }
    for (int i = 0; i < 2; ++i) {
      for (int h = 0; h < 2; ++h) {
        mbar_init(&sfull[i][h], 1);
        mbar_init(&pready[i][h], 4);
      }
      mbar_init(&pvdone[i], 1);
      mbar_init(&ofull[i], 1);
      mbar_init(&qready[i], 4);
    }
    mbar_init(&nready, 8);
    fence_barrier_init();
  }

  // ---- the CTA's range of units (group of query rows, tile of tokens)
  int64_t total = 0;
  for (int r = tid; r < a.B; r += PA_NT) total += pa_units(a, r);
  tc_before_sync();
  total = pa_sum(total, scr);
  tc_after_sync();
  const uint32_t tmem = tmem_base;
  const int64_t each = max((total + gridDim.x - 1) / (int64_t)gridDim.x, (int64_t)1);
  PaWalk<TREE> walk;
  const int64_t pos = blockIdx.x * each;
  walk.base = pos;
  walk.end = min(pos + each, total);
  walk.row = -1;
  walk.head = walk.mt = walk.tile0 = 0;
  walk.steps = walk.groups = walk.wides = 0;
  int4 join = make_int4(0, 0, 0, 0);
  if (pos < walk.end) {  // where it begins: rows' units counted up by all threads
    int64_t before = 0;
    for (int r0 = 0; r0 < a.B && walk.row < 0; r0 += PA_NT) {
      const int r = r0 + tid;
      const int64_t n = r < a.B ? pa_units(a, r) : 0;
      int64_t x = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      __syncthreads();
      if (lane == 31) scr[warp] = x;
      if (tid == 0) found = -1;
      __syncthreads();
      int64_t lo = before + x - n;
#pragma unroll
      for (int i = 0; i < PA_NT / 32; ++i) {
        if (i < warp) lo += scr[i];
        before += scr[i];
      }
      if (pos >= lo && pos < lo + n) {
        found = r;
        found_lo = lo;
      }
      __syncthreads();
      walk.row = found;
    }
    const AtRow rw = at_row<PA_ROWS / 8>(a, walk.row);
    const int64_t per_head = pa_units(a, walk.row) / a.heads, rel = pos - found_lo;
    walk.head = (int)(rel / per_head);
    int64_t u = rel - walk.head * per_head;
    walk.mt = rw.mt - 1;  // later groups see more: they come first
    for (int here; u >= (here = pa_tiles(a, rw, walk.mt) + pa_extra(a, rw, walk.mt)); --walk.mt) u -= here;
    const int extra = pa_extra(a, rw, walk.mt);
    walk.base = pos - u;
    walk.tile0 = (int)max(u - extra, (int64_t)0);
    // The first cut inside its group joins the pieces.
    const int64_t from = walk.base + extra;
    if (walk.tile0 > 0 && from >= ((int64_t)blockIdx.x - 1) * each)
      join = make_int4(walk.row, walk.mt * a.heads + walk.head, (int)((from + pa_tiles(a, rw, walk.mt) - 1) / each) - (int)blockIdx.x + 2, 0);
  }
  if (tid == 0) a.meta[blockIdx.x] = join;

  PaGroup g;
  if (warp < 8) {
    // ---- a thread per query row
    asm volatile("setmaxnreg.inc.sync.aligned.u32 144;");
    const int q = warp >> 2, r = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_at = tmem + 128 * q + lanes, o_at = tmem + 256 + 128 * q + lanes;
    uint32_t turns = 0;  // this stream's steps: their numbers choose the place of the scores
    for (; walk.get(a, g); walk.next(a, g)) {
      const bool narrow = g.narrow;
      const int tile = narrow ? 0 : q, rr = tile * 128 + r, ctx = g.ctx, start = g.start, see_last = g.see_last;
      const bool in = rr < g.rows;
      const int qi = in ? (g.mt * PA_ROWS + rr) / a.per : 0;
      const int qh = g.head * a.per + (in ? g.mt * PA_ROWS + rr - qi * a.per : 0);
      const int limit = !in ? 0 : TREE ? ctx : ctx + qi + 1;  // TREE: and what `shows` says
      const int at_place = TREE && in ? __ldg(&a.span[start + qi].x) : 0;
      auto shows = [&](int t) {  // new token t, below see_last
        const int2 b = __ldg(&a.span[start + t - ctx]);
        return in && (uint32_t)at_place - (uint32_t)b.x < (uint32_t)b.y;
      };
      float fq = fabsf(a.scale);
      if (!narrow || q == 0) {
        // Largest exponent of the row to 0 (bf16 to f16); the power of two goes into the row's factor.
        const uint16_t* src = reinterpret_cast<const uint16_t*>(a.q) + (int64_t)(start + qi) * a.q_st + (int64_t)qh * a.q_sh;
        float down = 1.0f;
        auto top_of = [&](uint32_t top, const uint4& v) {  // magnitudes of bf16 order as whole numbers do
          return __vmaxu2(__vmaxu2(top, v.x & 0x7fff7fffu), __vmaxu2(v.y & 0x7fff7fffu, __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu)));
        };
        auto factor = [&](uint32_t top) {
          top = max(top & 0xffffu, top >> 16);
          const int e = min(max((int)(top >> 7) - 127, -126), 126);
          down = __uint_as_float((uint32_t)(127 - e) << 23);
          fq *= __uint_as_float((uint32_t)(127 + e) << 23);
        };
        const uint32_t sign = a.scale < 0.0f ? 0x80008000u : 0u;  // scores are compared before they are scaled
        auto put = [&](int i, const uint4& v) {
          uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (DT == LSS_DTYPE_BF16) {
              const __half2 h = __floats2half2_rn(__uint_as_float(u[e] << 16) * down, __uint_as_float(u[e] & 0xffff0000u) * down);
              u[e] = *reinterpret_cast<const uint32_t*>(&h);
            }
            u[e] ^= sign;
          }
          *reinterpret_cast<uint4*>(qs + tile * OPB + pa_place(r, i)) = make_uint4(u[0], u[1], u[2], u[3]);
        };
        uint32_t top = 0;
        if (a.aligned) {
          uint4 v[CH];
#pragma unroll
          for (int i = 0; i < CH; ++i) v[i] = in ? __ldg(reinterpret_cast<const uint4*>(src) + i) : make_uint4(0, 0, 0, 0);
          if (DT == LSS_DTYPE_BF16) {
#pragma unroll
            for (int i = 0; i < CH; ++i) top = top_of(top, v[i]);
            factor(top);
          }
#pragma unroll
          for (int i = 0; i < CH; ++i) put(i, v[i]);
        } else {  // value by value, twice
          auto piece_of = [&](int i) {
            uint32_t u[4] = {0, 0, 0, 0};
            if (in) {
#pragma unroll
              for (int e = 0; e < 4; ++e) u[e] = (uint32_t)src[8 * i + 2 * e] | ((uint32_t)src[8 * i + 2 * e + 1] << 16);
            }
            return make_uint4(u[0], u[1], u[2], u[3]);
          };
          if (DT == LSS_DTYPE_BF16) {
#pragma unroll 1
            for (int i = 0; i < CH; ++i) top = top_of(top, piece_of(i));
            factor(top);
          }
#pragma unroll 1
          for (int i = 0; i < CH; ++i) put(i, piece_of(i));
        }
        if (narrow) row_factor[r] = fq;
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive_local(narrow ? &nready : &qready[q]);
      } else {  // the same rows
        __syncwarp();
        if (lane == 0) mbar_arrive_local(&nready);
        tc_wait(&nready, (walk.groups - walk.wides) & 1, &failed);
        fq = row_factor[r];
      }

      float m = -INFINITY, l = 0.0f, w = -INFINITY;
      // The first row of the warp sees least.
      const int see_warp = TREE ? ctx : ctx + (g.mt * PA_ROWS + tile * 128 + (warp & 3) * 32) / a.per + 1;
      const int first = narrow ? g.i0 + ((walk.steps ^ q) & 1) : g.i0, by = narrow ? 2 : 1, i1 = g.i1;
      for (int i = first; i < i1; i += by, ++turns) {
        const int half = turns & 1, at = i * PA_HT;
        tc_wait(&sfull[q][half], (turns >> 1) & 1, &failed);
        tc_after_sync();
        const uint32_t s_here = s_at + 64 * half;
        const float2* sc = sscale[(walk.steps + i - g.i0) & (PA_SC - 1)];
        // Without a mask the weights are first taken with the maxima as they are: if one, or a share of the softmax, is
        // too large for them (or NaN) they move and the weights are taken again.  A token's weight of V is 2^z,
        // z = s + log2(v scale) - W + 10; its share p = 2^(s - m) of the softmax differs by a factor of its part, so that
        // one exponential does for both: p = 2^z 2^(-shift).  Where the factor is far from 1 (a block of zeros has the
        // scale 2^-126) p would be lost: then p itself is taken.
        auto shift_of = [&](float ky) { return fminf((m == -INFINITY ? 0.0f : m) + ky - (w == -INFINITY ? 0.0f : w) + AT_BIAS, 126.0f); };
        const float4 k01 = *reinterpret_cast<const float4*>(sc), k23 = *reinterpret_cast<const float4*>(sc + 2);
        const float kx[4] = {k01.x, k01.z, k23.x, k23.z}, ky[4] = {k01.y, k01.w, k23.y, k23.w};
        const float least = fminf(fminf(ky[0], ky[1]), fminf(ky[2], ky[3]));
        bool over = at + PA_HT > see_warp || fminf(fminf(kx[0], kx[1]), fminf(kx[2], kx[3])) < 0.0f;
        const bool masked = over;
        over |= m == -INFINITY || shift_of(least) < -60.0f;
        float more = 0.0f;
        if (!__any_sync(0xffffffffu, over)) {
          uint32_t x[4][16], p[4][8];
#pragma unroll
          for (int g = 0; g < 4; ++g) tc_ld16(s_here + 16 * g, x[g]);
          tc_wait_ld();
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const float fg = fq * kx[g], add = ky[g] - w + AT_BIAS;
            float2 part = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
              const float2 y = fma2(make_float2(__uint_as_float(x[g][e]), __uint_as_float(x[g][e + 1])), make_float2(fg, fg), make_float2(add, add));
              const float2 v = make_float2(ex2(y.x), ex2(y.y));
              part = add2(part, v);
              const __half2 h = __floats2half2_rn(v.x, v.y);
              p[g][e / 2] = *reinterpret_cast<const uint32_t*>(&h);
            }
            const float sum = part.x + part.y, share = sum * ex2(-shift_of(ky[g]));
            over |= !(sum <= 32768.0f && share <= 1024.0f);  // 2^(AT_BIAS + AT_SLACK): each weight is an f16 below the largest
            more += share;
          }
          if (!__any_sync(0xffffffffu, over)) {
#pragma unroll
            for (int g = 0; g < 4; ++g) tc_st8(s_here + 8 * g, p[g]);  // over scores that have been read
          }
        }
        if (__any_sync(0xffffffffu, over)) {
          uint32_t x[4][16];
#pragma unroll
          for (int g = 0; g < 4; ++g) tc_ld16(s_here + 16 * g, x[g]);
          tc_wait_ld();
          uint32_t seen[2] = {0u, 0u};  // TREE, masked: the step's tokens that this row sees
          if (TREE && masked) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int t0 = at + 32 * h, old = min(max(limit - t0, 0), 32), upto = min(see_last - t0, 32);
              if (old > 0) seen[h] = 0xffffffffu >> (32 - old);
#pragma unroll 4
              for (int e = max(ctx - t0, 0); e < upto; ++e)
                if (shows(t0 + e)) seen[h] |= 1u << e;
            }
          }
          auto sees = [&](int e) { return TREE ? ((seen[e >> 5] >> (e & 31)) & 1u) != 0u : at + e < limit; };
          // Largest score, and largest weight of V.
          float top = -INFINITY, topw = -INFINITY;
          auto maxima = [&](auto mask_c) {
            constexpr bool with_mask = decltype(mask_c)::value;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              float t = -INFINITY;
#pragma unroll
              for (int e = 0; e < 16; ++e)
                if (!with_mask || sees(16 * g + e)) t = fmaxf(t, __uint_as_float(x[g][e]));
              if (with_mask && (kx[g] < 0.0f || (TREE ? ((seen[g >> 1] >> (16 * (g & 1))) & 0xffffu) == 0u : at + 16 * g >= limit))) continue;
              t = fmaxf(t * (fq * kx[g]), -FLT_MAX);  // -inf and NaN: seen, unlike what leaves m at -inf
              top = fmaxf(top, t);
              topw = fmaxf(topw, t + ky[g]);
            }
          };
          if (masked) maxima(std::true_type{}); else maxima(std::false_type{});
          if (__any_sync(0xffffffffu, top > m + AT_SLACK || topw > w + AT_SLACK)) {
            const float mn = fmaxf(m, top), wn = fmaxf(w, topw);
            l *= ex2(m - (mn == -INFINITY ? 0.0f : mn));
            const float shrink = ex2(w - (wn == -INFINITY ? 0.0f : wn));
            m = mn;
            w = wn;
            if (i > first) {  // the sums so far, once the products of the step before are in them
              tc_wait(&pvdone[q], (turns - 1) & 1, &failed);
              tc_after_sync();
#pragma unroll 1
              for (int d = 0; d < D; d += 16) {
                uint32_t o[16];
                tc_ld16(o_at + d, o);
                tc_wait_ld();
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * shrink);
                tc_st16(o_at + d, o);
              }
            }
          }
          const float mu = m == -INFINITY ? 0.0f : m;
          more = 0.0f;
          auto weights = [&](auto mask_c) {
            constexpr bool with_mask = decltype(mask_c)::value;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const float fg = fq * kx[g], gain = ex2(shift_of(ky[g]));
              uint32_t p[8];
#pragma unroll
              for (int e = 0; e < 16; e += 2) {
                float y0 = fmaf(__uint_as_float(x[g][e]), fg, -mu), y1 = fmaf(__uint_as_float(x[g][e + 1]), fg, -mu);
                if (with_mask) {
                  if (kx[g] < 0.0f || !sees(16 * g + e)) y0 = -INFINITY;
                  if (kx[g] < 0.0f || !sees(16 * g + e + 1)) y1 = -INFINITY;
                }
                const float p0 = ex2(y0), p1 = ex2(y1);
                more += p0 + p1;
                const __half2 v = __floats2half2_rn(p0 * gain, p1 * gain);
                p[e / 2] = *reinterpret_cast<const uint32_t*>(&v);
              }
              tc_st8(s_here + 8 * g, p);
            }
          };
          if (masked) weights(std::true_type{}); else weights(std::false_type{});
        }
        l += more;
        tc_wait_st();
        tc_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive_local(&pready[q][half]);
      }
      tc_wait(&ofull[q], walk.groups & 1, &failed);
      tc_after_sync();
      // Two streams of the same rows: the second one leaves its state, and its sums in the place of the queries, which no
      // product reads any more, four columns of all rows after the other.
      float4* other = reinterpret_cast<float4*>(qs);
      const bool both = narrow && g.i1 - g.i0 > 1;  // each has a step
      if (narrow) {
        if (q == 1) {
          tc_wait(&ofull[0], walk.groups & 1, &failed);
          state[0][r] = m;
          state[1][r] = l;
          state[2][r] = w;
          if (first < i1) {
#pragma unroll 2
            for (int i = 0; i < D; i += 16) {
              uint32_t x[16];
              tc_ld16(o_at + i, x);
              tc_wait_ld();
#pragma unroll
              for (int e = 0; e < 4; ++e)
                other[(i / 4 + e) * 128 + r] = make_float4(__uint_as_float(x[4 * e]), __uint_as_float(x[4 * e + 1]), __uint_as_float(x[4 * e + 2]), __uint_as_float(x[4 * e + 3]));
            }
          }
        }
        asm volatile("bar.sync 1, 256;" ::: "memory");
      }
      if (!narrow || q == 0) {
        float f0 = 1.0f, f1 = 0.0f;  // of this stream's sums and of the other's
        const bool mine = first < i1;  // a single step may be the other stream's
        if (narrow) {
          const float m1 = state[0][r], l1 = state[1][r], w1 = state[2][r];
          const float mn = fmaxf(m, m1), wn = fmaxf(w, w1), mu = mn == -INFINITY ? 0.0f : mn, wu = wn == -INFINITY ? 0.0f : wn;
          l = l * ex2(m - mu) + l1 * ex2(m1 - mu);
          f0 = ex2(w - wu);
          f1 = ex2(w1 - wu);
          m = mn;
          w = wn;
        }
        float* piece = a.part + ((size_t)blockIdx.x * 2 + (g.tile0 == 0 ? 1 : 0)) * pa_piece(D);
        const int* nans = nan_from[walk.groups & (NN - 1)];
        if (!g.whole && in) {  // a piece: its state as it is
          piece[rr] = m;
          piece[PA_ROWS + rr] = l;
          piece[2 * PA_ROWS + rr] = w;
        }
        if (!g.whole && tile == 0 && r < D) reinterpret_cast<int*>(piece + 3 * PA_ROWS + PA_ROWS * D)[r] = nans[r];
        const bool none = m == -INFINITY, bad = *(volatile int*)&failed, spoiled = bad || any_nan[walk.groups & (NN - 1)];
        const bool branches = TREE && branch_nan[walk.groups & (NN - 1)];
        const AtFactor fin(m, l, w);
        uint16_t* out = reinterpret_cast<uint16_t*>(a.out) + (int64_t)(start + qi) * a.o_st + (int64_t)qh * a.o_sh;
#pragma unroll 1
        for (int i = 0; i < D; i += 16) {
          uint32_t x[16];
          tc_ld16(o_at + i, x);
          tc_wait_ld();
          if (narrow && (both || !mine)) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float4 v = other[(i / 4 + e) * 128 + r];
              const float z[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
              for (int c = 0; c < 4; ++c) x[4 * e + c] = __float_as_uint(mine ? fmaf(z[c], f1, __uint_as_float(x[4 * e + c]) * f0) : z[c]);
            }
          }
          if (branches) {
#pragma unroll 1
            for (int t = max(ctx, g.tile0 * PA_KT); t < min(see_last, g.tile1 * PA_KT); ++t) {
              const int page = __ldg(a.table + g.row * a.table_stride + (t >> a.bs_shift));
              if (!shows(t) || (unsigned)page >= (unsigned)a.num_blocks) continue;
              const uint4 v = __ldg(reinterpret_cast<const uint4*>(
                  a.vc + (((((int64_t)page * a.heads + g.head) << a.bs_shift) + (t & ((1 << a.bs_shift) - 1))) * D + i)));
              const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
              for (int e = 0; e < 16; ++e)
                if (((u[e >> 2] >> (8 * (e & 3))) & 0x7fu) == 0x7fu) x[e] = 0x7fffffffu;
            }
          }
          if (!g.whole) {
            float* to = piece + 3 * PA_ROWS + rr * D + i;
            if (in)
#pragma unroll
              for (int e = 0; e < 16; e += 4)
                *reinterpret_cast<uint4*>(to + e) = bad ? make_uint4(NOWHERE, NOWHERE, NOWHERE, NOWHERE) : make_uint4(x[e], x[e + 1], x[e + 2], x[e + 3]);
          } else if (in) {
            uint32_t pk[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              float y[2];
#pragma unroll
              for (int z = 0; z < 2; ++z) {
                y[z] = none ? 0.0f : fin(__uint_as_float(x[2 * e + z]));
                if (spoiled && (bad || nans[i + 2 * e + z] < limit)) y[z] = __int_as_float(0x7fffffff);
              }
              pk[e] = at_pack<DT>(y[0], y[1]);
            }
            if (a.aligned) {
              reinterpret_cast<uint4*>(out + i)[0] = make_uint4(pk[0], pk[1], pk[2], pk[3]);
              reinterpret_cast<uint4*>(out + i)[1] = make_uint4(pk[4], pk[5], pk[6], pk[7]);
            } else {
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                out[i + 2 * e] = (uint16_t)pk[e];
                out[i + 2 * e + 1] = (uint16_t)(pk[e] >> 16);
              }
            }
          }
        }
        if (in && g.whole && a.lse) a.lse[(int64_t)(start + qi) * (a.heads * a.per) + qh] = none ? -INFINITY : (m + log2f(l)) * LN2;
      }
      if (narrow) asm volatile("bar.sync 1, 256;" ::: "memory");  // the other stream's sums have been read
      tc_before_sync();
    }
  } else if (warp < 16) {
    // ---- widen keys (warps 8 to 11) and values
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    const bool is_v = warp >= 12;
    const int ct = tid & 127;
    // Piece k of the thread: token + k PT, and the same 16 columns each time.
    constexpr int PT = 128 / (D / 16);
    const int cc = ct % (D / 16);
    const int token = ct / (D / 16) ^ (D > 64 && cc >= 4);  // lanes of the second panel take the neighbour: 8 lanes, 8 bank groups
    // Tokens PT apart lie PT lines apart, permuted alike.
    static_assert(PT % 8 == 0, "a thread's tokens are permuted alike");
    const uint32_t to0 = pa_place<PA_HT>(token, 2 * cc), to1 = pa_place<PA_HT>(token, 2 * cc + 1);
    const uint4* from0 = reinterpret_cast<const uint4*>(raw + (is_v ? RAWB : 0)) + token * (D / 16) + cc;
    unsigned char* into = is_v ? vsm : ksm;
    uint64_t *full = is_v ? vfull : kfull, *empty = is_v ? vempty : kempty;
    for (; walk.get(a, g); walk.next(a, g)) {
      int* nans = nan_from[walk.groups & (NN - 1)];
      if (is_v) {
        if (ct < D) nans[ct] = NOWHERE;
        if (ct == 0) any_nan[walk.groups & (NN - 1)] = branch_nan[walk.groups & (NN - 1)] = 0;
        asm volatile("bar.sync 3, 128;" ::: "memory");
      }
      for (int i = g.i0; i < g.i1; ++i) {
        const uint32_t n = walk.steps + i - g.i0, rst = n % RS, st = n % OP;
        tc_wait(&rfull[is_v][rst], (n / RS) & 1, &failed);
        const uint4* from = from0 + rst * (2 * RAWB / 16);
        uint4 v[PIECES];
#pragma unroll
        for (int k = 0; k < PIECES; ++k) v[k] = from[k * 128];
        if (is_v) {
          const uint32_t there = parts[n & (PA_SC - 1)];
          const bool cut = i * PA_HT + PA_HT > g.see_all || there != 15u;
          if (cut) {  // nothing of parts and tokens that are not there, and no NaN
#pragma unroll
            for (int k = 0; k < PIECES; ++k) {
              const int t = token + k * PT;
              if (!((there >> (t >> 4)) & 1u) || i * PA_HT + t >= g.see_last) v[k] = make_uint4(0, 0, 0, 0);
              uint32_t u[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
              uint32_t any = 0;
#pragma unroll
              for (int e = 0; e < 4; ++e) any |= (u[e] & 0x7f7f7f7fu) + 0x01010101u;  // a byte of 0x7f carries into its sign
              if (any & 0x80808080u) {
                any_nan[walk.groups & (NN - 1)] = 1;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const uint32_t nan = __vcmpeq4(u[e] & 0x7f7f7f7fu, 0x7f7f7f7fu);
                  for (int z = 0; z < 4; ++z)
                    if ((nan >> (8 * z)) & 1u) {
                      if (TREE && i * PA_HT + t >= g.ctx) branch_nan[walk.groups & (NN - 1)] = 1;
                      else atomicMin(&nans[cc * 16 + 4 * e + z], i * PA_HT + t);
                    }
                  u[e] &= ~nan;
                }
                v[k] = make_uint4(u[0], u[1], u[2], u[3]);
              }
            }
          }
        }
        if (n >= OP) tc_wait(&empty[st], (n / OP - 1) & 1, &failed);
        unsigned char* to = into + st * STB;
#pragma unroll
        for (int k = 0; k < PIECES; ++k) {
          const uint32_t u[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
          *reinterpret_cast<uint4*>(to + k * PT * 128 + to0) = make_uint4(f16_of_e4m3(u[0]), f16_of_e4m3(u[0] >> 16), f16_of_e4m3(u[1]), f16_of_e4m3(u[1] >> 16));
          *reinterpret_cast<uint4*>(to + k * PT * 128 + to1) = make_uint4(f16_of_e4m3(u[2]), f16_of_e4m3(u[2] >> 16), f16_of_e4m3(u[3]), f16_of_e4m3(u[3] >> 16));
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive_local(&full[st]);
          mbar_arrive_local(&rempty[is_v][rst]);
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    if (warp < 18) {
      // ---- issue a stream's products: scores are two of its steps ahead of the weighted values
      constexpr uint32_t is = tc_idesc(false, PA_HT), io = tc_idesc(false, D) | (1u << 16);  // values: columns lie together
      const int q = warp - 16;
      const uint32_t s_at = tmem + 128 * q, o_at = tmem + 256 + 128 * q;
      uint32_t turns = 0;
      for (; walk.get(a, g); walk.next(a, g)) {
        const bool narrow = g.narrow;
        const int first = narrow ? g.i0 + ((walk.steps ^ q) & 1) : g.i0, by = narrow ? 2 : 1;
        const uint32_t q0 = tc_desc_lo(saddr(qs + (narrow ? 0 : q) * OPB));
        if (narrow) tc_wait(&nready, (walk.groups - walk.wides) & 1, &failed);
        else tc_wait(&qready[q], walk.wides & 1, &failed);
        auto score = [&](int i, uint32_t turn) {
          const uint32_t n = walk.steps + i - g.i0, st = n % OP, half = turn & 1;
          const bool ok = tc_wait(&kfull[st], (n / OP) & 1, &failed);
          tc_after_sync();
          __syncwarp();
          if (tc_elect()) {
            const uint32_t k0 = tc_desc_lo(saddr(ksm + st * STB));
            if (ok) {
#pragma unroll
              for (int s = 0; s < D / 16; ++s)
                tc_mma_ss(s_at + 64 * half, q0 + ((s >> 2) * (128 * 128) + (s & 3) * 32) / 16, TC_DESC_HI, k0 + ((s >> 2) * (PA_HT * 128) + (s & 3) * 32) / 16,
                          TC_DESC_HI, is, s > 0);
            }
            tc_commit(&sfull[q][half]);
            tc_commit(&kempty[st]);
            if (narrow) mbar_arrive_local(&kempty[st]);  // for the other stream
          }
          __syncwarp();
        };
        auto weigh = [&](int i, uint32_t turn) {
          const uint32_t n = walk.steps + i - g.i0, st = n % OP, half = turn & 1;
          bool ok = tc_wait(&vfull[st], (n / OP) & 1, &failed);
          ok = tc_wait(&pready[q][half], (turn >> 1) & 1, &failed) && ok;
          tc_after_sync();
          __syncwarp();
          if (tc_elect()) {
            // panels of 64 columns are 8 KB apart, groups of 8 tokens 1 KB
            const uint32_t v0 = ((saddr(vsm + st * STB) >> 4) & 0x3fffu) | ((PA_HT * 128u >> 4) << 16);
            if (ok) {
#pragma unroll
              for (int s = 0; s < PA_HT / 16; ++s)
                tc_mma_ts(o_at, s_at + 64 * half + 8 * s, v0 + s * (2048 / 16), TC_DESC_HI, io, i > first || s > 0);
            }
            tc_commit(&pvdone[q]);
            tc_commit(&vempty[st]);
            if (narrow) mbar_arrive_local(&vempty[st]);
          }
          __syncwarp();
        };
        for (int j = 0; j < 2; ++j)
          if (first + j * by < g.i1) score(first + j * by, turns + j);
#pragma unroll 1
        for (int i = first; i < g.i1; i += by, ++turns) {
          weigh(i, turns);
          if (i + 2 * by < g.i1) score(i + 2 * by, turns + 2);
        }
        if (tc_elect()) tc_commit(&ofull[q]);
        __syncwarp();
      }
    } else {
      // ---- issue the copies, of the keys (warp 18) and of the values: lanes 0 to 3 a part of 16 tokens each; block ids of
      // 32 parts at a time, one per lane.  The scales of both go with the keys: the softmax needs them first.
      const int bsm = (1 << a.bs_shift) - 1, part = lane & 3;
      const bool is_v = warp == 19;
      const uint8_t* codes = is_v ? a.vc : a.kc;
      const float* scales = lane & 4 ? a.vs : a.ks;
      for (; walk.get(a, g); walk.next(a, g)) {
        const int32_t* trow = a.table + g.row * a.table_stride;
        auto load_ids = [&](int from) {  // of parts [from, from + 32)
          const int t = (from + lane) * 16;
          const int page = t < g.see_last ? __ldg(trow + (t >> a.bs_shift)) : -1;
          return (unsigned)page < (unsigned)a.num_blocks ? page : -1;
        };
        int at = g.i0 * 4, ids = load_ids(at), ids_next = load_ids(at + 32);
        auto page_of = [&](int i) {  // of this lane's part of step i: called for steps in order
          if (i * 4 - at >= 32) {
            at += 32;
            ids = ids_next;
            ids_next = load_ids(at + 32);
          }
          return __shfl_sync(0xffffffffu, ids, i * 4 + part - at);
        };
        auto scale_of = [&](int page) { return page >= 0 && !is_v && lane < 8 ? __ldg(scales + (int64_t)page * a.heads + g.head) : -1.0f; };
        int page = page_of(g.i0);
        float scale = scale_of(page);
        for (int i = g.i0; i < g.i1; ++i) {
          const uint32_t n = walk.steps + i - g.i0, rst = n % RS;
          const int page_now = page;
          const float scale_now = scale;
          if (i + 1 < g.i1) {
            page = page_of(i + 1);
            scale = scale_of(page);
          }
          bool ok = n < RS || tc_wait(&rempty[is_v][rst], (n / RS - 1) & 1, &failed);
          ok = ok && !*(volatile int*)&failed;
          const bool mine = lane < 4 && page_now >= 0;
          const uint32_t there = __ballot_sync(0xffffffffu, mine);
          if (is_v) {
            if (lane == 0) parts[n & (PA_SC - 1)] = there;
          } else if (lane < 8) {
            float2* sc = &sscale[n & (PA_SC - 1)][part];
            if (lane < 4) sc->x = scale_now;
            else sc->y = page_now >= 0 ? lg2(scale_now) : -INFINITY;
          }
          __syncwarp();
          if (lane == 0) mbar_expect_tx(&rfull[is_v][rst], ok ? __popc(there) * 16 * D : 0);
          __syncwarp();
          if (mine && ok) {
            const int t = i * PA_HT + part * 16;
            bulk_g2s(raw + rst * 2 * RAWB + (is_v ? RAWB : 0) + part * 16 * D, codes + ((((int64_t)page_now * a.heads + g.head) << a.bs_shift) + (t & bsm)) * D, 16 * D,
                     &rfull[is_v][rst]);
          }
        }
      }
    }
  }
  __syncwarp();
  tc_before_sync();
  __syncthreads();
  tc_after_sync();
  if (*(volatile int*)&failed) {  // products and copies may still run: they get a quarter of a second
    const long long t0 = clock64();
    while (clock64() - t0 < T4_WAIT / 4) __nanosleep(1000);
    __syncthreads();
  }
  if (warp == 0) tc_free(tmem, 512);
}

// Adds up the pieces of a group that was cut, the last one of the CTA before and the first ones of this
// CTA and those after it; 32 rows per CTA.
template <int D, int DT, bool TREE>
__global__ void __launch_bounds__(256) lss_attend_tc_join_kernel(AttendArgs a) {
  pdl_wait();
  const int cta = blockIdx.x / (PA_ROWS / 32), r0 = blockIdx.x % (PA_ROWS / 32) * 32;
  const int4 me = a.meta[cta];
  if (me.z == 0) return;
  const AtRow rw = at_row<PA_ROWS / 8>(a, me.x);
  const int head = me.y % a.heads, mt = me.y / a.heads;
  const int rows_here = min(PA_ROWS, rw.n * a.per - mt * PA_ROWS);
  auto piece = [&](int i) { return a.part + (size_t)(i == 0 ? (cta - 1) * 2 + 1 : (cta + i - 1) * 2) * pa_piece(D); };
  for (int x = threadIdx.x; x < 32 * (D / 4); x += 256) {
    const int rr = r0 + x / (D / 4), d = x % (D / 4) * 4;
    if (rr >= rows_here) break;
    float m = -INFINITY, w = -INFINITY;
    int nan[4] = {INT32_MAX, INT32_MAX, INT32_MAX, INT32_MAX};
    for (int i = 0; i < me.z; ++i) {
      const float* p = piece(i);
      m = fmaxf(m, p[rr]);
      w = fmaxf(w, p[2 * PA_ROWS + rr]);
      const int4 n4 = *reinterpret_cast<const int4*>(p + 3 * PA_ROWS + PA_ROWS * D + d);
      nan[0] = min(nan[0], n4.x);
      nan[1] = min(nan[1], n4.y);
      nan[2] = min(nan[2], n4.z);
      nan[3] = min(nan[3], n4.w);
    }
    const float mu = m == -INFINITY ? 0.0f : m, wu = w == -INFINITY ? 0.0f : w;
    float l = 0.0f, o[4] = {};
    for (int i = 0; i < me.z; ++i) {
      const float* p = piece(i);
      l += p[PA_ROWS + rr] * ex2(p[rr] - mu);
      const float f = ex2(p[2 * PA_ROWS + rr] - wu);
      const float4 v = *reinterpret_cast<const float4*>(p + 3 * PA_ROWS + rr * D + d);
      o[0] += v.x * f;
      o[1] += v.y * f;
      o[2] += v.z * f;
      o[3] += v.w * f;
    }
    const bool none = m == -INFINITY;  // it sees nothing
    const AtFactor f(m, l, w);
    const int r2 = mt * PA_ROWS + rr, qi = r2 / a.per, qh = head * a.per + r2 - qi * a.per;
    const int limit = rw.len - rw.n + qi + 1;
    const int64_t tok = a.starts[me.x] + qi;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      o[e] = none ? 0.0f : f(o[e]);
      if (nan[e] < limit) o[e] = __int_as_float(0x7fffffff);
    }
    const uint32_t y0 = at_pack<DT>(o[0], o[1]), y1 = at_pack<DT>(o[2], o[3]);
    uint16_t* out = reinterpret_cast<uint16_t*>(a.out) + tok * a.o_st + (int64_t)qh * a.o_sh + d;
    out[0] = (uint16_t)y0;
    out[1] = (uint16_t)(y0 >> 16);
    out[2] = (uint16_t)y1;
    out[3] = (uint16_t)(y1 >> 16);
    if (a.lse && d == 0) a.lse[tok * (a.heads * a.per) + qh] = none ? -INFINITY : (m + log2f(l)) * LN2;
  }
}

}  // namespace lss
