// lss_attend.cuh — softmax attention of a step's queries over a paged key/value cache of 8-bit
// values (e4m3) with one scale per block and key head.
#pragma once

#include "lss_kvcache.cuh"

namespace lss {

// The weights of V are held in f16 times 2^AT_BIAS; running maxima move when a score exceeds them by
// more than AT_SLACK (powers of two: 2^(AT_BIAS + AT_SLACK) stays below the largest f16).
constexpr float AT_BIAS = 10.0f, AT_SLACK = 5.0f;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

// Shape of the kernel for a head dimension, query rows per group (8 NQ) and tiles a step (TP): warps per
// CTA (one CTA per SM), stages of the copy ring per warp.  Registers set the warps (queries and sums take
// 6 NQ D / 16 of them), the shared memory the stages.  D = 128, 8 rows: two tiles a step on 12 warps give each
// warp more to do between its waits (1.1 GB of contexts of up to 16,000 tokens: 223 -> 212 us); one on 16 warps
// starts more groups at once (512 rows of 64 to 300 tokens: 75 us against 92).  At D = 256 the registers are full with one
// tile; D = 64 has not been built with two.
template <int D, int NQ, int TP> struct AtCfg;
template <> struct AtCfg<64, 1, 1> { static constexpr int NW = 16, ST = 6; };
template <> struct AtCfg<64, 2, 1> { static constexpr int NW = 16, ST = 6; };
template <> struct AtCfg<64, 4, 1> { static constexpr int NW = 12, ST = 8; };
template <> struct AtCfg<128, 1, 1> { static constexpr int NW = 16, ST = 3; };
template <> struct AtCfg<128, 1, 2> { static constexpr int NW = 12, ST = 4; };
template <> struct AtCfg<128, 2, 1> { static constexpr int NW = 12, ST = 4; };
template <> struct AtCfg<128, 4, 1> { static constexpr int NW = 8, ST = 6; };
template <> struct AtCfg<256, 1, 1> { static constexpr int NW = 8, ST = 3; };
template <> struct AtCfg<256, 2, 1> { static constexpr int NW = 8, ST = 3; };
// Floats of one piece in the workspace: m, l, W of its rows, then the sums.
__host__ __device__ constexpr int at_piece(int D, int NQ) { return 8 * NQ * (3 + D); }

// From this many tokens on, rows of fewer queries pay for the start and end of a group in tensor memory, and those of 16 queries more
// (launch_attend_rows).
static constexpr int AT_LONG = 2560;
__host__ __device__ constexpr int at_long_more(int D) { return D == 128 ? 640 : 1024; }

struct AttendArgs {
  const void* q;
  int64_t q_st, q_sh;  // strides in elements: token, head
  void* out;
  int64_t o_st, o_sh;
  float* lse;          // [T][q_heads] or NULL
  const uint8_t* kc;   // [num_blocks][heads][block_size][D]
  const uint8_t* vc;
  const float* ks;     // [num_blocks][heads]
  const float* vs;
  int num_blocks, heads, per, bs_shift;
  const int32_t* table;
  int64_t table_stride;
  int width;
  const int32_t* starts;
  const int32_t* granted;
  const int32_t* lens;
  const int2* span;    // [T]: place in its tree's pre-order and size of its branch (kernels with TREE)
  int B, T;
  float scale;         // softmax scale times log2(e)
  int aligned;         // q and out rows start on 16-byte boundaries
  // Which rows of the batch are this launch's: all, those for tensor memory, or the others.  For tensor memory are rows of
  // rows_any query rows per key head and more, and long ones from rows_long on.
  int side;  // 0, 1, 2
  int rows_any, rows_long, long_more;
  int fused;           // the grid is one cluster, which joins its own pieces
  int4* meta;          // [workers]: row, group, pieces (0: nothing to join)
  float* part;         // [workers][2][at_piece]: a warp's first piece, its last one
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 8x8 matrix of 16-bit values, two of a row per lane, transposed across the warp.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t f16_of_e4m3(uint32_t two) {  // the two low bytes
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)two));
  return r;
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ float lds32f(uint32_t a) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}

// Where the 16-byte piece `cc` of a token's columns lies in a tile of 16 tokens (one panel of PC
// columns): pieces are permuted inside 128-byte lines so that the 8 lanes that one wide shared
// load serves at a time read 8 different bank groups, for K (2 tokens x 4 column groups) and for
// V (2 column groups x 4 token pairs) alike.
template <int PC>
__device__ __forceinline__ uint32_t at_offset(int token, int cc) {
  if (PC == 128) return (uint32_t)(token * 128 + ((cc ^ (token & 7)) << 4));
  const int line = token >> 1;
  return (uint32_t)(line * 128 + ((((token & 1) * 4 + cc) ^ ((line << 1) & 7)) << 4));
}

// A row's share of the work: groups of 8 NQ query rows per key head, tiles of 16 tokens.  Rows whose
// numbers do not fit (more new tokens than tokens, outside the table or the batch's tokens), and those of another
// launch, have none.
struct AtRow {
  int n, len, nt, mt;
};
template <int NQ>
__device__ __forceinline__ AtRow at_row(const AttendArgs& a, int r) {
  AtRow w;
  w.n = a.granted[r];
  w.len = a.lens[r];
  const int s = a.starts[r];
  const bool ok = w.n > 0 && w.n <= w.len && w.len <= ((int64_t)a.width << a.bs_shift) && s >= 0 && (int64_t)s + w.n <= a.T;
  const int64_t rows = (int64_t)w.n * a.per;
  const bool tensor = rows >= a.rows_any || (rows >= a.rows_long && w.len >= (rows < a.rows_long + 16 ? AT_LONG : a.long_more));
  if (!ok || (a.side && tensor != (a.side == 1))) w.n = 0;
  w.nt = w.n > 0 ? (w.len + 15) >> 4 : 0;
  w.mt = w.n > 0 ? (int)(((int64_t)w.n * a.per + 8 * NQ - 1) / (8 * NQ)) : 0;
  return w;
}

// One finished value row segment: n values x[i] * f to the 16-bit output.
template <int DT>
__device__ __forceinline__ uint32_t at_pack(float x0, float x1) {
  if (DT == LSS_DTYPE_BF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(x0, x1);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  const __half2 v = __floats2half2_rn(x0, x1);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// What turns a row's sums into its result, 2^(W - AT_BIAS - m) / l, as f times g: with the smallest scales of V
// the power alone would be flushed to zero.
struct AtFactor {
  float f, g;
  __device__ __forceinline__ AtFactor(float m, float l, float w) {
    const float e = w - AT_BIAS - m;
    const bool low = e < -64.0f;
    f = ex2(low ? e + 64.0f : e) / l;
    g = low ? 5.42101086242752217e-20f : 1.0f;  // 2^-64
  }
  __device__ __forceinline__ float operator()(float x) const { return x * f * g; }
};

// Adds up `n` pieces (at p(i), laid out as in the workspace) of one group and writes the result: the
// output where `last`, else a piece at `dst`.  Threads t0, t0 + nth, ... share the elements.
template <int D, int DT, int NQ, class PieceAt>
__device__ __forceinline__ void at_join(const AttendArgs& a, PieceAt piece_at, int n, bool last, float* dst, int row,
                                        int item, int t0, int nth) {
  constexpr int R = 8 * NQ;
  const AtRow rw = at_row<NQ>(a, row);
  const int head = item / rw.mt, mt = item - head * rw.mt;
  const int rows_here = min(R, rw.n * a.per - mt * R);
  for (int x = t0; x < rows_here * (D / 4); x += nth) {
    const int rr = x / (D / 4), d = (x % (D / 4)) * 4;
    float m = -INFINITY, w = -INFINITY;
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
      const float* p = piece_at(i);
      m = fmaxf(m, p[rr]);
      w = fmaxf(w, p[2 * R + rr]);
    }
    const float mu = m == -INFINITY ? 0.0f : m, wu = w == -INFINITY ? 0.0f : w;
    float l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
      const float* p = piece_at(i);
      const float pl = p[R + rr];
      const float4 v = *reinterpret_cast<const float4*>(p + 3 * R + rr * D + d);
      l += pl * ex2(p[rr] - mu);
      const float f = ex2(p[2 * R + rr] - wu);
      if (pl != 0.0f) {  // else it saw nothing, or another one holds it: nothing was written there
        o.x += v.x * f;
        o.y += v.y * f;
        o.z += v.z * f;
        o.w += v.w * f;
      }
    }
    if (!last) {
      if (d == 0) {
        dst[rr] = m;
        dst[R + rr] = l;
        dst[2 * R + rr] = w;
      }
      *reinterpret_cast<float4*>(dst + 3 * R + rr * D + d) = o;
      continue;
    }
    const AtFactor f(m, l, w);
    const bool none = m == -INFINITY;  // it sees nothing
    const uint32_t y0 = none ? 0u : at_pack<DT>(f(o.x), f(o.y)), y1 = none ? 0u : at_pack<DT>(f(o.z), f(o.w));
    const int r2 = mt * R + rr, qi = r2 / a.per, qh = head * a.per + r2 - qi * a.per;
    const int64_t tok = a.starts[row] + qi;
    uint16_t* out = reinterpret_cast<uint16_t*>(a.out) + tok * a.o_st + (int64_t)qh * a.o_sh + d;
    if (a.aligned) {
      *reinterpret_cast<uint2*>(out) = make_uint2(y0, y1);
    } else {
      out[0] = (uint16_t)y0;
      out[1] = (uint16_t)(y0 >> 16);
      out[2] = (uint16_t)y1;
      out[3] = (uint16_t)(y1 >> 16);
    }
    if (a.lse && d == 0) a.lse[tok * (a.heads * a.per) + qh] = none ? -INFINITY : (m + log2f(l)) * LN2;
  }
}

// The group that `worker` joins: its pieces are the last one of the warp before, then the first ones of this
// warp and those after it.  Inside a CTA they are added up already, in the place of the first of them; so what
// counts is the one before, the first warp of each CTA that follows, and the last warp, whose first piece may
// stand alone.
template <int D, int DT, int NQ, int TP>
__device__ __forceinline__ void at_join_cut(const AttendArgs& a, int64_t worker, const int4& me, int t0, int nth) {
  constexpr int NW = AtCfg<D, NQ, TP>::NW;
  constexpr int64_t PS = at_piece(D, NQ);
  const int64_t end = worker + me.z - 2, cta = (worker + NW - 1) / NW;
  const int ctas = end >= cta * NW ? (int)(end / NW - cta) + 1 : 0;
  const bool extra = end % NW != 0;
  at_join<D, DT, NQ>(a, [&](int i) {
    const int64_t at = i == 0 ? (worker - 1) * 2 + 1 : i <= ctas ? (cta + i - 1) * NW * 2 : end * 2;
    return a.part + at * PS;
  }, 1 + ctas + extra, true, nullptr, me.x, me.y, t0, nth);
}

// o = sum_t p_t v_t,  p = softmax_t(c q . k_t) over the tokens t up to the query's own position.
//
// Work: for each row and key head, the queries that share it (`per` heads times the row's new
// tokens) in groups of 8 NQ, times the row's tokens in tiles of 16.  These units, in that order, are
// cut into equal ranges, one per warp, whatever the lengths are: every warp streams its own tiles
// through its own copy ring and keeps its own running softmax, with no barrier between warps.
// Ranges that end inside a group leave pieces: those of the CTA's warps are added up in shared memory,
// those of several CTAs by lss_attend_join_kernel, always in order; where the work fits one cluster
// (`fused`), behind a cluster barrier instead, which saves a launch.
//
// Arithmetic: with keys and values as the 16-row operand of mma.m16n8k16 (f16 operands, f32 sums),
// S^T = K Q^T and O^T = V^T P^T need no padding for 8 query rows, and the weights turn from result to
// operand by one 8x8 transpose per 8 tokens.  e4m3 values are exact in f16; bf16 queries are scaled by a
// power of two per row so that they are exact in f16 down to 2^-24 of the row's largest.  The column
// order inside a product is free, so each lane takes its values where they lie (32 consecutive
// columns of two tokens for K, 16 of four tokens for V) and no operand is shuffled between lanes.
// Scales of the blocks: that of K multiplies the score, that of V joins the exponent of the weight
// that multiplies V, w_t = 2^(s_t + log2(v scale) - W + 10), with a running maximum W of its own.
// Both maxima may lag behind by 2^5 (one vote per tile instead of reductions); the weights are rounded
// to f16 (2^-11 relative, no more than the result's own rounding) and keep that precision down to
// 2^-24 of the largest one.  The sum of the softmax is f32.
//
// Measured at D = 128, 8 key heads: 1.1 GB of contexts of 50 to 16,000 tokens for 64 single queries of 32 heads
// 212 us (5.2 TB/s, 0.81 of the copy rate), 733 MB of three contexts of 90,000 to 131,000 140 us (226 and 146 with other
// work between the calls); with queries as the 16-row operand (half of it padding) and reductions for every tile it was
// 268 and 200 us.  The first at D = 64 138 us (0.62 of the copy rate), at D = 256 400 us (0.86).
// Bound by HBM (2 D bytes per token and head) when a row has few queries, by the tensor pipe and the
// widening of the codes when it has many (they share it 8 NQ rows at a time).
//
// With TREE the row's new tokens are the nodes of a tree (parents before children): a query sees the tokens before
// them and, of them, those in whose branch it lies.  With a node's place in the pre-order and the size of its branch
// that is one unsigned comparison per new token, 0 <= place(query) - place(token) < size(token), in the tiles that hold
// new tokens; all others take the same path as without.  As parents come first, the last token that a group of
// queries can see, and with it the split of the work, is that of the causal form.
template <int D, int DT, int NQ, int TP, bool TREE>
__global__ void __launch_bounds__(AtCfg<D, NQ, TP>::NW * 32, 1) lss_attend_kernel(AttendArgs a) {
  constexpr int NW = AtCfg<D, NQ, TP>::NW, ST = AtCfg<D, NQ, TP>::ST, NTH = NW * 32, R = 8 * NQ;
  constexpr int PC = D < 128 ? D : 128, NP = D / PC;  // columns per panel, panels
  constexpr int SP = PC / 16;                         // 16-column steps per panel
  constexpr int STAGE = 32 * D + 16;                  // K tile, V tile, two scales
  constexpr int PIECE = at_piece(D, NQ);
  constexpr int PD = ST / TP;                         // steps in the ring
  static_assert(ST % TP == 0 && PD > 1, "a step is computed while another one is under way");
  static_assert(PIECE * 4 <= ST * STAGE, "a piece lies in its warp's ring");
  extern __shared__ __align__(128) unsigned char at_sm[];
  __shared__ int64_t scr[NW];
  __shared__ int64_t w_excl[NW];
  __shared__ int w_row[NW];
  __shared__ int4 w_last[NW];  // a warp's last piece: row (-1: complete), group, first tile, pieces to join
  __shared__ int w_end[NW];    // whether it ends its group
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, c = lane & 3;

  // ---- this warp's range of units
  auto units_of = [&](int r) -> int64_t {
    const AtRow w = at_row<NQ>(a, r);
    return (int64_t)a.heads * w.mt * w.nt;
  };
  int64_t total = 0;
  const int64_t u0 = tid < a.B ? units_of(tid) : 0;
  {
    int64_t mine = u0;
    for (int r = tid + NTH; r < a.B; r += NTH) mine += units_of(r);
    mine = warp_allreduce(mine, [](int64_t p, int64_t q) { return p + q; });
    if (lane == 0) scr[warp] = mine;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NW; ++i) total += scr[i];
  }
  const int64_t workers = (int64_t)gridDim.x * NW;
  const int64_t each = max((total + workers - 1) / workers, (int64_t)1);
  const int64_t first_w = (int64_t)blockIdx.x * NW;
  int64_t base = 0;
  for (int r0 = 0; r0 < a.B; r0 += NTH) {
    const int r = r0 + tid;
    const int64_t u = r0 == 0 ? u0 : (r < a.B ? units_of(r) : 0);
    int64_t x = u;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) scr[warp] = x;
    __syncthreads();
    int64_t before = base;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      if (i < warp) before += scr[i];
      base += scr[i];
    }
    const int64_t lo = before + x - u, hi = before + x;
    if (hi > first_w * each && lo < (first_w + NW) * each) {
#pragma unroll
      for (int i = 0; i < NW; ++i) {
        const int64_t s = (first_w + i) * each;
        if (s >= lo && s < hi) {
          w_row[i] = r;
          w_excl[i] = lo;
        }
      }
    }
  }
  __syncthreads();
  const int64_t worker = first_w + warp;
  int64_t pos = worker * each;
  const int64_t end = min(pos + each, total);
  int row = pos < end ? w_row[warp] : 0;
  int64_t excl = pos < end ? w_excl[warp] : 0;
  const uint32_t ring = saddr(at_sm) + (uint32_t)warp * (ST * STAGE);
  float* own = reinterpret_cast<float*>(at_sm + (size_t)warp * (ST * STAGE));  // the last piece, at the end
  int4 last = make_int4(-1, 0, 0, 0);
  int last_end = 0;
  int4 join = make_int4(0, 0, 0, 0);

  // Where the lane's first 16 bytes of a tile go; the ones 512 bytes on follow by rule (at_offset).
  const uint32_t copy_to = (uint32_t)(lane % (D / 16) / (PC / 16)) * (16 * PC) + at_offset<PC>(lane / (D / 16), lane % (D / 16) % (PC / 16));

  while (pos < end) {
    const AtRow rw = at_row<NQ>(a, row);
    const int64_t rel = pos - excl;
    const int item = (int)(rel / rw.nt);
    const int tile0 = (int)(rel - (int64_t)item * rw.nt);
    const int tile1 = (int)min((int64_t)rw.nt, (int64_t)tile0 + (end - pos));
    const int head = item / rw.mt, mt = item - head * rw.mt;
    const int start = a.starts[row], ctx = rw.len - rw.n;
    const int rows_here = min(R, rw.n * a.per - mt * R);
    // Tokens that the first and the last query of the group see.
    const int see_first = TREE ? ctx : ctx + mt * R / a.per + 1;
    const int see_last = ctx + (mt * R + rows_here - 1) / a.per + 1;
    const int tend = min(tile1, (see_last + 15) >> 4);
    auto sees = [&](int rr) { return rr < rows_here ? ctx + (mt * R + rr) / a.per + 1 : 0; };
    // TREE: place of a row's query in its tree; what a token shows, and to whom (below see_last only).
    auto place = [&](int rr) { return rr < rows_here ? __ldg(&a.span[start + (mt * R + rr) / a.per].x) : -1; };
    auto branch = [&](int token) {
      if (token < ctx) return make_int2(INT32_MIN, -1);  // any place is in it
      return token < see_last ? __ldg(&a.span[start + token - ctx]) : make_int2(0, 0);
    };
    auto within = [](int at, const int2& b) { return (uint32_t)at - (uint32_t)b.x < (uint32_t)b.y; };
    int at_place[NQ][2];
    if constexpr (TREE) {
#pragma unroll
      for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
        for (int e = 0; e < 2; ++e) at_place[nq][e] = place(8 * nq + 2 * c + e);
    }

    // ---- copies: block ids of 32 tiles at a time, one per lane
    const int32_t* trow = a.table + row * a.table_stride;
    int ids_base = tile0;
    auto load_ids = [&](int from) {
      const int t = from + lane;
      return t < tend ? trow[(t << 4) >> a.bs_shift] : 0;
    };
    int ids = load_ids(tile0), ids_next = load_ids(tile0 + 32);
    uint32_t bad = 0;  // bit s: the tile in stage s lies in no block of the cache
    auto issue = [&](int t, int s) {
      if (t < tend) {
        if (t - ids_base >= 32) {
          ids_base = t;
          ids = ids_next;
          ids_next = load_ids(t + 32);
        }
        int page = __shfl_sync(0xffffffffu, ids, t - ids_base);
        const bool wrong = (unsigned)page >= (unsigned)a.num_blocks;
        bad = wrong ? bad | (1u << s) : bad & ~(1u << s);
        page = wrong ? 0 : page;
        const int64_t ph = (int64_t)page * a.heads + head;
        const int64_t off = ((ph << a.bs_shift) + ((t << 4) & ((1 << a.bs_shift) - 1))) * D + lane * 16;
        const uint8_t* ksrc = a.kc + off;
        const uint8_t* vsrc = a.vc + off;
        const uint32_t dst = ring + (uint32_t)s * STAGE;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          const uint32_t to = D == 64 ? copy_to + 512 * i : D == 128 ? (copy_to ^ ((i & 1) << 6)) + 512 * i : (copy_to ^ ((i & 3) << 5)) + 256 * i;
          cp_async16(dst + to, ksrc + 512 * i);
          cp_async16(dst + 16 * D + to, vsrc + 512 * i);
        }
        if (lane < 2) {
          const float* src = (lane == 0 ? a.ks : a.vs) + ph;
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst + 32 * D + 4 * lane), "l"(src) : "memory");
        }
      }
      cp_async_commit();
    };
    __syncwarp();
#pragma unroll
    for (int s = 0; s < (PD - 1) * TP; ++s) issue(tile0 + s, s);

    // ---- queries: lane (g, c) holds row g of each eight, its columns; factors of rows 2c, 2c + 1
    uint32_t qf[NQ][NP * SP][2];
    float fq[NQ][2];
#pragma unroll
    for (int nq = 0; nq < NQ; ++nq) {
      const int rr = mt * R + 8 * nq + g;
      const bool in = 8 * nq + g < rows_here;
      const int qi = in ? rr / a.per : 0;
      const int64_t at = in ? (int64_t)(start + qi) * a.q_st + (int64_t)(head * a.per + rr - qi * a.per) * a.q_sh : 0;
      const uint16_t* src = reinterpret_cast<const uint16_t*>(a.q) + at;
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        const uint16_t* s = src + p * PC + c * (PC / 4);
#pragma unroll
        for (int j = 0; j < SP; j += 2) {
          uint4 v = make_uint4(0, 0, 0, 0);
          if (in) {
            if (a.aligned) {
              v = __ldg(reinterpret_cast<const uint4*>(s + 4 * j));
            } else {
              uint32_t* u = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
              for (int q = 0; q < 4; ++q) u[q] = (uint32_t)s[4 * j + 2 * q] | ((uint32_t)s[4 * j + 2 * q + 1] << 16);
            }
          }
          qf[nq][p * SP + j][0] = v.x;
          qf[nq][p * SP + j][1] = v.y;
          qf[nq][p * SP + j + 1][0] = v.z;
          qf[nq][p * SP + j + 1][1] = v.w;
        }
      }
      float f = 1.0f;
      if (DT == LSS_DTYPE_BF16) {
        float amax = 0.0f;
#pragma unroll
        for (int j = 0; j < NP * SP; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float x0 = fabsf(__uint_as_float(qf[nq][j][e] << 16)), x1 = fabsf(__uint_as_float(qf[nq][j][e] & 0xffff0000u));
            if (x0 <= FLT_MAX) amax = fmaxf(amax, x0);
            if (x1 <= FLT_MAX) amax = fmaxf(amax, x1);
          }
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        // Largest exponent to 0: values become less than 2 in magnitude.
        const int e = min(max((int)(__float_as_uint(amax) >> 23) - 127, -126), 126);
        const float down = __uint_as_float((uint32_t)(127 - e) << 23);
        f = __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
        for (int j = 0; j < NP * SP; ++j)
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const __half2 v = __floats2half2_rn(__uint_as_float(qf[nq][j][q] << 16) * down, __uint_as_float(qf[nq][j][q] & 0xffff0000u) * down);
            qf[nq][j][q] = *reinterpret_cast<const uint32_t*>(&v);
          }
      }
      f *= a.scale;
      fq[nq][0] = __shfl_sync(0xffffffffu, f, 8 * c);
      fq[nq][1] = __shfl_sync(0xffffffffu, f, 8 * c + 4);
    }

    // ---- running state of rows 2c, 2c + 1 of each eight: maximum m and sum l (of this lane's tokens) of
    // the softmax, maximum W of the weights of V, sums o
    float m[NQ][2], l[NQ][2], w[NQ][2];
    float o[NP * SP][NQ][4];
#pragma unroll
    for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        m[nq][e] = w[nq][e] = -INFINITY;
        l[nq][e] = 0.0f;
      }
#pragma unroll
    for (int i = 0; i < NP * SP; ++i)
#pragma unroll
      for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
        for (int q = 0; q < 4; ++q) o[i][nq][q] = 0.0f;

    uint32_t stage = 0, fill = (PD - 1) * TP;
    for (int t0 = tile0; t0 < tend; t0 += TP) {
      // TP tiles a step: the places of the step before are free once all lanes are here.
      __syncwarp();
#pragma unroll
      for (int u = 0; u < TP; ++u) {
        issue(t0 + (PD - 1) * TP + u, (int)fill);
        fill = fill + 1 == ST ? 0 : fill + 1;
      }
      cp_async_wait_group<(PD - 1) * TP>();
      __syncwarp();
      uint32_t kt[TP];
      bool wrong[TP], masked[TP];
      float lv[TP], f[TP][NQ][2], s[TP][NQ][4];
      bool any_masked = false;
#pragma unroll
      for (int u = 0; u < TP; ++u) {
        kt[u] = ring + stage * STAGE;
        wrong[u] = ((bad >> stage) & 1u) || t0 + u >= tend;
        stage = stage + 1 == ST ? 0 : stage + 1;
        masked[u] = wrong[u] || ((t0 + u) << 4) + 16 > see_first;
        any_masked |= masked[u];
        const float kscale = lds32f(kt[u] + 32 * D);
        lv[u] = lg2(lds32f(kt[u] + 32 * D + 4));
        if (wrong[u]) lv[u] = 0.0f;  // what lies there may be anything
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq) {
          f[u][nq][0] = fq[nq][0] * kscale;
          f[u][nq][1] = fq[nq][1] * kscale;
        }
      }

      // scores: rows of the product are tokens g and g + 8
#pragma unroll
      for (int u = 0; u < TP; ++u)
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[u][nq][e] = 0.0f;
#pragma unroll
      for (int p = 0; p < NP; ++p) {
#pragma unroll
        for (int i = 0; i < SP / 4; ++i) {
#pragma unroll
          for (int u = 0; u < TP; ++u) {
            const uint4 x = lds128(kt[u] + p * (16 * PC) + at_offset<PC>(g, c * (SP / 4) + i));
            const uint4 y = lds128(kt[u] + p * (16 * PC) + at_offset<PC>(g + 8, c * (SP / 4) + i));
            const uint32_t xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint32_t ka[4] = {f16_of_e4m3(xw[j]), f16_of_e4m3(yw[j]), f16_of_e4m3(xw[j] >> 16), f16_of_e4m3(yw[j] >> 16)};
#pragma unroll
              for (int nq = 0; nq < NQ; ++nq) mma_f16(s[u][nq], ka, qf[nq][p * SP + 4 * i + j][0], qf[nq][p * SP + 4 * i + j][1]);
            }
          }
        }
      }
      // log2 of a token's share of the softmax over 2^m (y), and of its weight of V (z)
      uint32_t pb[TP][NQ][2];
      float y[TP][NQ][4], z[TP][NQ][4];
      bool over = false;
      uint32_t hidden = 0;  // TREE: bit 4 (u NQ + nq) + e
      if (TREE && any_masked) {
#pragma unroll
        for (int u = 0; u < TP; ++u)
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const int2 b = branch(((t0 + u) << 4) + g + 8 * q);
#pragma unroll
            for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
              for (int e = 0; e < 2; ++e)
                if (wrong[u] || !within(at_place[nq][e], b)) hidden |= 1u << (4 * (u * NQ + nq) + 2 * q + e);
          }
      }
      auto exponents = [&]() {
#pragma unroll
        for (int u = 0; u < TP; ++u)
#pragma unroll
          for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float mu = m[nq][e & 1], add = lv[u] - w[nq][e & 1] + AT_BIAS;
              y[u][nq][e] = fmaf(s[u][nq][e], f[u][nq][e & 1], -mu);
              z[u][nq][e] = fmaf(s[u][nq][e], f[u][nq][e & 1], add);
            }
        if (any_masked) {
#pragma unroll
          for (int u = 0; u < TP; ++u)
#pragma unroll
            for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (TREE ? (hidden >> (4 * (u * NQ + nq) + e)) & 1u : wrong[u] || ((t0 + u) << 4) + g + 8 * (e >> 1) >= sees(8 * nq + 2 * c + (e & 1)))
                  y[u][nq][e] = z[u][nq][e] = -INFINITY;
        }
      };
      exponents();
#pragma unroll
      for (int u = 0; u < TP; ++u)
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
          for (int e = 0; e < 4; ++e) over |= !(y[u][nq][e] <= AT_SLACK && z[u][nq][e] <= AT_BIAS + AT_SLACK);  // NaN too: -inf less a maximum of -inf
      if (__any_sync(0xffffffffu, over)) {  // the first step, and where the maxima move
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float top = -INFINITY, topw = -INFINITY;
#pragma unroll
            for (int u = 0; u < TP; ++u) {
              float tu = -INFINITY;
#pragma unroll
              for (int q = 0; q < 2; ++q) {
                const bool see = !any_masked || (TREE ? !((hidden >> (4 * (u * NQ + nq) + 2 * q + e)) & 1u)
                                                      : !wrong[u] && ((t0 + u) << 4) + g + 8 * q < sees(8 * nq + 2 * c + e));
                // A score of -inf is above "none seen": maxima of what is seen are finite at least, so that such a
                // score has no weight beside others, and no sum at all alone (0 / 0 at the end).
                if (see) tu = fmaxf(tu, fmaxf(s[u][nq][2 * q + e] * f[u][nq][e], -FLT_MAX));
              }
              top = fmaxf(top, tu);
              topw = fmaxf(topw, tu + lv[u]);
            }
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) {
              top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
              topw = fmaxf(topw, __shfl_xor_sync(0xffffffffu, topw, x));
            }
            const float mn = fmaxf(m[nq][e], top), wn = fmaxf(w[nq][e], topw);
            l[nq][e] *= ex2(m[nq][e] - (mn == -INFINITY ? 0.0f : mn));
            const float shrink = ex2(w[nq][e] - (wn == -INFINITY ? 0.0f : wn));
            m[nq][e] = mn;
            w[nq][e] = wn;
#pragma unroll
            for (int i = 0; i < NP * SP; ++i) {
              o[i][nq][e] *= shrink;
              o[i][nq][2 + e] *= shrink;
            }
          }
        exponents();
      }
#pragma unroll
      for (int u = 0; u < TP; ++u)
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq) {
          l[nq][0] += ex2(y[u][nq][0]) + ex2(y[u][nq][2]);
          l[nq][1] += ex2(y[u][nq][1]) + ex2(y[u][nq][3]);
          const __half2 lo = __floats2half2_rn(ex2(z[u][nq][0]), ex2(z[u][nq][1])), hi = __floats2half2_rn(ex2(z[u][nq][2]), ex2(z[u][nq][3]));
          pb[u][nq][0] = transpose8(*reinterpret_cast<const uint32_t*>(&lo));
          pb[u][nq][1] = transpose8(*reinterpret_cast<const uint32_t*>(&hi));
        }

      // weights times values: rows of the product are columns of V
#pragma unroll
      for (int u = 0; u < TP; ++u)
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        uint32_t vw[4][PC / 32];  // tokens 2c, 2c+1, 2c+8, 2c+9; the lane's columns
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int token = 2 * c + (r & 1) + 8 * (r >> 1);
          if constexpr (PC == 128) {
            const uint4 v = lds128(kt[u] + 16 * D + p * (16 * PC) + at_offset<PC>(token, g));
            vw[r][0] = v.x;
            vw[r][1] = v.y;
            vw[r][2] = v.z;
            vw[r][3] = v.w;
          } else {
            const uint2 v = lds64(kt[u] + 16 * D + at_offset<PC>(token, g >> 1) + (g & 1) * 8);
            vw[r][0] = v.x;
            vw[r][1] = v.y;
          }
        }
        if (masked[u]) {
          if (wrong[u] || ((t0 + u) << 4) + 16 > see_last) {  // tokens that no query of the group sees: 0 times what lies there may be NaN
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (wrong[u] || ((t0 + u) << 4) + 2 * c + (r & 1) + 8 * (r >> 1) >= see_last) {
#pragma unroll
                for (int i = 0; i < PC / 32; ++i) vw[r][i] = 0u;
              }
          }
          // Tokens that only some queries of the group see: a NaN among their values belongs to
          // those alone, so it leaves the product below and is added where it is seen.
          uint32_t found = 0u;
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int i = 0; i < PC / 32; ++i) found |= __vcmpeq4(vw[r][i] & 0x7f7f7f7fu, 0x7f7f7f7fu);
          if (__any_sync(0xffffffffu, found != 0u)) {
#pragma unroll
            for (int i = 0; i < PC / 32; ++i) {
              uint32_t one[4];  // 1 (0x38) where a value is NaN
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const uint32_t nan = __vcmpeq4(vw[r][i] & 0x7f7f7f7fu, 0x7f7f7f7fu);
                one[r] = nan & 0x38383838u;
                vw[r][i] &= ~nan;
              }
#pragma unroll
              for (int q = 0; q < 2; ++q) {
                const uint32_t sel = q == 0 ? 0x5140u : 0x7362u;
                const uint32_t n0 = __byte_perm(one[0], one[1], sel), n1 = __byte_perm(one[2], one[3], sel);
                const uint32_t na[4] = {f16_of_e4m3(n0), f16_of_e4m3(n0 >> 16), f16_of_e4m3(n1), f16_of_e4m3(n1 >> 16)};
#pragma unroll
                for (int nq = 0; nq < NQ; ++nq) {
                  const int lim = sees(8 * nq + g), tk = ((t0 + u) << 4) + 2 * c;
                  const int at = TREE ? place(8 * nq + g) : 0;
                  auto seen = [&](int t) { return TREE ? within(at, branch(t)) : t < lim; };
                  float count[4] = {};
                  mma_f16(count, na, (seen(tk) ? 0x3c00u : 0u) | (seen(tk + 1) ? 0x3c000000u : 0u),
                          (seen(tk + 8) ? 0x3c00u : 0u) | (seen(tk + 9) ? 0x3c000000u : 0u));
#pragma unroll
                  for (int e = 0; e < 4; ++e)
                    if (count[e] > 0.0f) o[p * SP + 2 * i + q][nq][e] = __int_as_float(0x7fffffff);
                }
              }
            }
          }
        }
#pragma unroll
        for (int i = 0; i < PC / 32; ++i)
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const uint32_t sel = q == 0 ? 0x5140u : 0x7362u;
            const uint32_t t0 = __byte_perm(vw[0][i], vw[1][i], sel), t1 = __byte_perm(vw[2][i], vw[3][i], sel);
            const uint32_t va[4] = {f16_of_e4m3(t0), f16_of_e4m3(t0 >> 16), f16_of_e4m3(t1), f16_of_e4m3(t1 >> 16)};
#pragma unroll
            for (int nq = 0; nq < NQ; ++nq) mma_f16(o[p * SP + 2 * i + q][nq], va, pb[u][nq][0], pb[u][nq][1]);
          }
      }
    }  // the next tile's __syncwarp lets its place be written again
    asm volatile("cp.async.wait_all;" ::: "memory");

#pragma unroll
    for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[nq][e] += __shfl_xor_sync(0xffffffffu, l[nq][e], x);
    // Lane (g, c) holds rows 2c and 2c + 1 of each eight, columns p * PC + g * PC / 8 + 2 i + (0, 1): the
    // sums o[p * SP + i][nq][e] and [2 + e].
    const bool whole = tile0 == 0 && tile1 == rw.nt;
    const bool is_last = pos + (tile1 - tile0) == end;
    float* dst = is_last ? own : a.part + (worker * 2) * PIECE;  // a first piece that the warp goes on from
    __syncwarp();
#pragma unroll
    for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int rr = 8 * nq + 2 * c + e;
        if (rr < rows_here) {
          if (whole) {
            const int r2 = mt * R + rr, qi = r2 / a.per, qh = head * a.per + r2 - qi * a.per;
            const bool none = m[nq][e] == -INFINITY;
            const AtFactor f(m[nq][e], l[nq][e], w[nq][e]);
            uint16_t* out = reinterpret_cast<uint16_t*>(a.out) + (int64_t)(start + qi) * a.o_st + (int64_t)qh * a.o_sh;
#pragma unroll
            for (int p = 0; p < NP; ++p)
#pragma unroll
              for (int i = 0; i < SP; i += 4) {
                uint32_t pk[4];
#pragma unroll
                for (int q = 0; q < 4; ++q)
                  pk[q] = none ? 0u : at_pack<DT>(f(o[p * SP + i + q][nq][e]), f(o[p * SP + i + q][nq][2 + e]));
                uint16_t* d = out + p * PC + g * (PC / 8) + 2 * i;
                if (a.aligned) {
                  *reinterpret_cast<uint4*>(d) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
                } else {
#pragma unroll
                  for (int q = 0; q < 4; ++q) {
                    d[2 * q] = (uint16_t)pk[q];
                    d[2 * q + 1] = (uint16_t)(pk[q] >> 16);
                  }
                }
              }
            if (a.lse && g == 0)
              a.lse[(int64_t)(start + qi) * (a.heads * a.per) + qh] = none ? -INFINITY : (m[nq][e] + log2f(l[nq][e])) * LN2;
          } else {
            if (g == 0) {
              dst[rr] = m[nq][e];
              dst[R + rr] = l[nq][e];
              dst[2 * R + rr] = w[nq][e];
            }
#pragma unroll
            for (int p = 0; p < NP; ++p)
#pragma unroll
              for (int i = 0; i < SP; i += 2)
                *reinterpret_cast<float4*>(dst + 3 * R + rr * D + p * PC + g * (PC / 8) + 2 * i) =
                    make_float4(o[p * SP + i][nq][e], o[p * SP + i][nq][2 + e], o[p * SP + i + 1][nq][e], o[p * SP + i + 1][nq][2 + e]);
          }
        }
      }
    if (!whole) {
      if (is_last) {
        last = make_int4(row, item, tile0, 0);
        last_end = tile1 == rw.nt;
      }
      if (tile0 > 0) {  // the first cut inside its group joins the pieces
        const int64_t from = pos - tile0;
        if (from >= (worker - 1) * each) join = make_int4(row, item, (int)((from + rw.nt - 1) / each - worker + 2), 0);
      }
    }
    pos += tile1 - tile0;
    if (pos < end && pos - excl >= (int64_t)a.heads * rw.mt * rw.nt) {
      excl += (int64_t)a.heads * rw.mt * rw.nt;
      do ++row; while (row < a.B - 1 && at_row<NQ>(a, row).n == 0);
    }
  }

  // ---- last pieces of consecutive warps that belong to one group are added up here; the sum stands
  // in the place of the first of them, and the others' places are marked empty
  if (lane == 0) {
    w_last[warp] = last;
    w_end[warp] = last_end;
  }
  __syncthreads();
  for (int w0 = 0; w0 < NW;) {
    const int4 p = w_last[w0];
    int w1 = w0 + 1;
    if (p.x >= 0) {
      while (w1 < NW && w_last[w1].x == p.x && w_last[w1].y == p.y) ++w1;
      const bool done = p.z == 0 && w_end[w1 - 1];
      float* dst = a.part + ((first_w + w0) * 2 + (p.z == 0 ? 1 : 0)) * PIECE;
      at_join<D, DT, NQ>(a, [&](int i) { return reinterpret_cast<const float*>(at_sm + (size_t)(w0 + i) * (ST * STAGE)); }, w1 - w0,
                         done, dst, p.x, p.y, tid, NTH);
      if (done) {
        if (warp > w0 && warp < w1) join.z = 0;
      } else if (warp > w0 && warp < w1) {
        float* mine = a.part + worker * 2 * PIECE;
        if (lane < R) {
          mine[lane] = mine[2 * R + lane] = -INFINITY;
          mine[R + lane] = 0.0f;
        }
      }
    }
    w0 = w1;
  }
  if (a.fused) {
    __threadfence();
    cg::this_cluster().sync();
    if (lane == 0) w_last[warp] = join;
    __syncthreads();
    for (int i = 0; i < NW; ++i)
      if (w_last[i].z > 0) at_join_cut<D, DT, NQ, TP>(a, first_w + i, w_last[i], tid, NTH);
  } else if (lane == 0) {
    a.meta[worker] = join;
  }
}

// Adds up the pieces of the groups that were cut between CTAs: one CTA per warp of the first kernel,
// most with nothing to do.
template <int D, int DT, int NQ, int TP, bool TREE>
__global__ void __launch_bounds__(256) lss_attend_join_kernel(AttendArgs a) {
  pdl_wait();
  const int4 me = a.meta[blockIdx.x];
  if (me.z > 0) at_join_cut<D, DT, NQ, TP>(a, blockIdx.x, me, threadIdx.x, 256);
}

}  // namespace lss
