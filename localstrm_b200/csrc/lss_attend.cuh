// lss_attend.cuh — softmax attention of a step's queries over a paged key/value cache of 8-bit
// values (e4m3) with one scale per block and key head.
#pragma once

#include "lss_kvcache.cuh"

namespace lss {

constexpr int AT_MIN_UNITS = 4;   // tiles of 16 tokens that a warp takes at least
constexpr float AT_BIAS = 14.0f;  // the weights of V are held times 2^14 in f16 (see below)
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

// Shape of the kernel for one head dimension: warps per CTA (one CTA per SM), stages of the
// copy ring per warp.
template <int D> struct AtCfg;
template <> struct AtCfg<64> { static constexpr int NW = 16, ST = 6; };
template <> struct AtCfg<128> { static constexpr int NW = 12, ST = 4; };
template <> struct AtCfg<256> { static constexpr int NW = 8, ST = 3; };

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
  int B, T;
  float scale;         // softmax scale times log2(e)
  int aligned;         // q and out rows start on 16-byte boundaries
  int4* meta;          // [workers]: row, item, pieces (0: nothing to join)
  float* part;         // [workers][2][48 + 16 * D]: m, l, w of 16 rows, then the sums
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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

// A row's share of the work.  Invalid rows (more new tokens than tokens, outside the table or the
// batch's tokens) have none.
struct AtRow {
  int n, len, nt, mt;
};
__device__ __forceinline__ AtRow at_row(const AttendArgs& a, int r) {
  AtRow w;
  w.n = a.granted[r];
  w.len = a.lens[r];
  const int s = a.starts[r];
  const bool ok = w.n > 0 && w.n <= w.len && w.len <= ((int64_t)a.width << a.bs_shift) && s >= 0 && (int64_t)s + w.n <= a.T;
  if (!ok) w.n = 0;
  w.nt = w.n > 0 ? (w.len + 15) >> 4 : 0;
  w.mt = w.n > 0 ? (int)(((int64_t)w.n * a.per + 15) >> 4) : 0;
  return w;
}

// o = sum_t p_t v_t,  p = softmax_t(c q . k_t) over the tokens t up to the query's own position.
//
// Work: for each row and key head, the queries that share it (`per` heads times the row's new
// tokens) in groups of 16, times the row's tokens in tiles of 16.  These units, in that order, are
// cut into equal ranges, one per warp, whatever the lengths are: every warp streams its own tiles
// through its own copy ring and keeps its own running softmax, with no barrier between warps.  A
// range that ends inside a group writes its state to the workspace and lss_attend_join_kernel adds
// the pieces up in order.
//
// Arithmetic: a group of 16 tokens is two 16x8 products with q and D/8 with the weights
// (mma.m16n8k16, f16 operands, f32 sums).  e4m3 values are exact in f16; bf16 queries are scaled by a
// power of two per row so that they are exact in f16 down to 2^-24 of the row's largest.  The column
// order inside a product is free, so each lane takes its values where they lie (32 consecutive
// columns of one token for K, 16 of four tokens for V) and no fragment is shuffled between lanes.
// Scales of the blocks: that of K multiplies the score, that of V joins the exponent of the weight
// that multiplies V, w_t = f 2^(s_t + e - W + 14) for a scale f 2^e, with a running maximum W of its own.
// The weights are rounded to f16 (2^-11 relative, no more than the result's own rounding); with the
// factor 2^14 they keep that precision down to 2^-28 of the largest one.  The sum of the softmax is f32.
//
// Bound by HBM (2 D bytes per token and head) when a row has few queries: 16 query rows per value
// read is far below what the tensor pipe can do.
template <int D, int DT>
__global__ void __launch_bounds__(AtCfg<D>::NW * 32, 1) lss_attend_kernel(AttendArgs a) {
  constexpr int NW = AtCfg<D>::NW, ST = AtCfg<D>::ST, NTH = NW * 32;
  constexpr int PC = D < 128 ? D : 128, NP = D / PC;  // columns per panel, panels
  constexpr int SP = PC / 16;                         // products of 16 columns per panel
  constexpr int NB = PC / 8;                          // products of 8 output columns per panel
  constexpr int STAGE = 32 * D + 16;                  // K tile, V tile, two scales
  extern __shared__ __align__(128) unsigned char at_sm[];
  __shared__ int64_t scr[NW];
  __shared__ int64_t w_excl[NW];
  __shared__ int w_row[NW];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, c = lane & 3;

  // ---- this warp's range of units
  auto units_of = [&](int r) -> int64_t {
    const AtRow w = at_row(a, r);
    return (int64_t)a.heads * w.mt * w.nt;
  };
  int64_t mine = 0, total;
  const int64_t u0 = tid < a.B ? units_of(tid) : 0;
  mine = u0;
  for (int r = tid + NTH; r < a.B; r += NTH) mine += units_of(r);
  if (tid < NW) w_row[tid] = -1;
  {
    int64_t x = warp_allreduce(mine, [](int64_t p, int64_t q) { return p + q; });
    if (lane == 0) scr[warp] = x;
    __syncthreads();
    total = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) total += scr[i];
  }
  const int64_t workers = (int64_t)gridDim.x * NW;
  int64_t each = (total + workers - 1) / workers;
  if (each < AT_MIN_UNITS) each = AT_MIN_UNITS;
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
    if (u > 0) {
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
  if (pos >= end) {
    if (lane == 0) a.meta[worker] = make_int4(0, 0, 0, 0);
    return;
  }
  int row = w_row[warp];
  int64_t excl = w_excl[warp];
  const uint32_t ring = saddr(at_sm) + (uint32_t)warp * (ST * STAGE);
  bool wrote_meta = false;

  while (pos < end) {
    const AtRow rw = at_row(a, row);
    const int64_t rel = pos - excl;
    const int item = (int)(rel / rw.nt);
    const int tile0 = (int)(rel - (int64_t)item * rw.nt);
    const int tile1 = (int)min((int64_t)rw.nt, (int64_t)tile0 + (end - pos));
    const int head = item / rw.mt, mt = item - head * rw.mt;
    const int start = a.starts[row], ctx = rw.len - rw.n;
    const int rows_here = min(16, rw.n * a.per - mt * 16);
    // Tokens that the first and the last query of the group see.
    const int see_first = ctx + mt * 16 / a.per + 1;
    const int see_last = ctx + (mt * 16 + rows_here - 1) / a.per + 1;
    const int tend = min(tile1, (see_last + 15) >> 4);

    // ---- queries: rows g and g + 8 of the group, the lane's columns
    uint32_t qf[NP * SP][4];
    float qs[2];
    int limit[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int rr = mt * 16 + g + 8 * h;
      const bool in = g + 8 * h < rows_here;
      const int qi = in ? rr / a.per : 0;
      limit[h] = in ? ctx + qi + 1 : 0;
      const int64_t at = in ? (int64_t)(start + qi) * a.q_st + (int64_t)(head * a.per + rr - qi * a.per) * a.q_sh : 0;
      const uint16_t* src = reinterpret_cast<const uint16_t*>(a.q) + at;
      uint32_t raw[NP * SP][2];
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
          raw[p * SP + j][0] = v.x;
          raw[p * SP + j][1] = v.y;
          raw[p * SP + j + 1][0] = v.z;
          raw[p * SP + j + 1][1] = v.w;
        }
      }
      float f = 1.0f;
      if (DT == LSS_DTYPE_BF16) {
        float amax = 0.0f;
#pragma unroll
        for (int j = 0; j < NP * SP; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float x0 = fabsf(__uint_as_float(raw[j][e] << 16)), x1 = fabsf(__uint_as_float(raw[j][e] & 0xffff0000u));
            if (x0 <= FLT_MAX) amax = fmaxf(amax, x0);
            if (x1 <= FLT_MAX) amax = fmaxf(amax, x1);
          }
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        // Largest exponent to 0: values become at most 2 in magnitude.
        const int e = min(max((int)(__float_as_uint(amax) >> 23) - 127, -126), 126);
        const float down = __uint_as_float((uint32_t)(127 - e) << 23);
        f = __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
        for (int j = 0; j < NP * SP; ++j)
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const __half2 v = __floats2half2_rn(__uint_as_float(raw[j][q] << 16) * down, __uint_as_float(raw[j][q] & 0xffff0000u) * down);
            raw[j][q] = *reinterpret_cast<const uint32_t*>(&v);
          }
      }
      qs[h] = f * a.scale;
#pragma unroll
      for (int j = 0; j < NP * SP; ++j) {
        qf[j][h] = raw[j][0];
        qf[j][2 + h] = raw[j][1];
      }
    }

    // ---- running state: softmax maximum m and sum l, maximum W of the weights of V, sums o
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f}, w[2] = {-INFINITY, -INFINITY};
    float o[NP * NB][4];
#pragma unroll
    for (int i = 0; i < NP * NB; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) o[i][q] = 0.0f;

    // Block ids of 32 tiles at a time, one per lane.
    const int32_t* trow = a.table + row * a.table_stride;
    int ids = 0, ids_base = tile0;
    auto load_ids = [&](int from) {
      const int t = from + lane;
      return t < tend ? trow[(t << 4) >> a.bs_shift] : 0;
    };
    ids = load_ids(tile0);
    uint32_t bad = 0;  // bit s: the tile in stage s lies in no block of the cache
    auto issue = [&](int t, int s) {
      if (t < tend) {
        if (t - ids_base >= 32) {
          ids_base = t;
          ids = load_ids(t);
        }
        int page = __shfl_sync(0xffffffffu, ids, t - ids_base);
        const bool wrong = page < 0 || page >= a.num_blocks;
        bad = wrong ? bad | (1u << s) : bad & ~(1u << s);
        page = wrong ? 0 : page;
        const int64_t ph = (int64_t)page * a.heads + head;
        const int64_t off = ((ph << a.bs_shift) + ((t << 4) & ((1 << a.bs_shift) - 1))) * D;
        const uint32_t dst = ring + (uint32_t)s * STAGE;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          const int q = lane + 32 * i, token = q / (D / 16), cc = q % (D / 16);
          const uint32_t to = (uint32_t)(cc / (PC / 16)) * (16 * PC) + at_offset<PC>(token, cc % (PC / 16));
          cp_async16(dst + to, a.kc + off + 16 * q);
          cp_async16(dst + 16 * D + to, a.vc + off + 16 * q);
        }
        if (lane < 2) {
          const float* src = lane == 0 ? a.ks + ph : a.vs + ph;
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst + 32 * D + 4 * lane), "l"(src) : "memory");
        }
      }
      cp_async_commit();
    };
    __syncwarp();
#pragma unroll
    for (int s = 0; s < ST - 1; ++s) issue(tile0 + s, s);
    int stage = 0, fill = ST - 1;

    for (int t = tile0; t < tend; ++t) {
      cp_async_wait_group<ST - 2>();
      __syncwarp();
      issue(t + ST - 1, fill);
      fill = fill + 1 == ST ? 0 : fill + 1;
      const uint32_t kt = ring + (uint32_t)stage * STAGE, vt = kt + 16 * D;
      const bool wrong = (bad >> stage) & 1u;
      stage = stage + 1 == ST ? 0 : stage + 1;
      const float kscale = lds32f(kt + 32 * D), vscale = lds32f(kt + 32 * D + 4);

      // scores
      float s[2][4] = {};
#pragma unroll
      for (int n8 = 0; n8 < 2; ++n8) {
        const int token = 8 * n8 + g;
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          uint32_t kw[SP];
#pragma unroll
          for (int i = 0; i < SP / 4; ++i) {
            const uint4 v = lds128(kt + p * (16 * PC) + at_offset<PC>(token, c * (SP / 4) + i));
            kw[4 * i] = v.x;
            kw[4 * i + 1] = v.y;
            kw[4 * i + 2] = v.z;
            kw[4 * i + 3] = v.w;
          }
#pragma unroll
          for (int j = 0; j < SP; ++j) mma_f16(s[n8], qf[p * SP + j], f16_of_e4m3(kw[j]), f16_of_e4m3(kw[j] >> 16));
        }
      }
      const bool masked = wrong || (t << 4) + 16 > see_first;
      const float f0 = qs[0] * kscale, f1 = qs[1] * kscale;
#pragma unroll
      for (int n8 = 0; n8 < 2; ++n8) {
        s[n8][0] *= f0;
        s[n8][1] *= f0;
        s[n8][2] *= f1;
        s[n8][3] *= f1;
      }
      if (masked) {
#pragma unroll
        for (int n8 = 0; n8 < 2; ++n8)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (wrong || (t << 4) + 8 * n8 + 2 * c + (e & 1) >= limit[e >> 1]) s[n8][e] = -INFINITY;
      }
      // vscale = vf * 2^lv; a scale that is no normal number stays in vf as far as it can.
      const int vexp = (int)((__float_as_uint(vscale) >> 23) & 255u);
      const float lv = (float)(min(max(vexp, 1), 254) - 127);
      const float vf = vexp == 255 ? vscale
                       : vexp == 0 ? vscale * 8.507059173023462e37f
                                   : __uint_as_float((__float_as_uint(vscale) & 0x807fffffu) | 0x3f800000u);
      uint32_t pa[4];
      bool moved = false;
      float shrink[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float top = fmaxf(fmaxf(s[0][2 * h], s[0][2 * h + 1]), fmaxf(s[1][2 * h], s[1][2 * h + 1]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float mn = fmaxf(m[h], top), wn = fmaxf(w[h], top + lv);
        const float mu = mn == -INFINITY ? 0.0f : mn, wu = wn == -INFINITY ? 0.0f : wn;
        l[h] *= ex2(m[h] - mu);
        shrink[h] = ex2(w[h] - wu);
        moved |= wn != w[h];
        m[h] = mn;
        w[h] = wn;
        const float add = lv - wu + AT_BIAS;
        float p4[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = s[e >> 1][2 * h + (e & 1)];
          l[h] += ex2(x - mu);
          p4[e] = ex2(x + add) * vf;
        }
        const __half2 lo = __floats2half2_rn(p4[0], p4[1]), hi = __floats2half2_rn(p4[2], p4[3]);
        pa[h] = *reinterpret_cast<const uint32_t*>(&lo);
        pa[2 + h] = *reinterpret_cast<const uint32_t*>(&hi);
      }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int i = 0; i < NP * NB; ++i) {
          o[i][0] *= shrink[0];
          o[i][1] *= shrink[0];
          o[i][2] *= shrink[1];
          o[i][3] *= shrink[1];
        }
      }

      // weights times values
      const bool tail = wrong || (t << 4) + 16 > see_last;  // tokens that no query of the group sees
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        uint32_t vw[4][PC / 32];  // tokens 2c, 2c+1, 2c+8, 2c+9; the lane's columns
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int token = 2 * c + (r & 1) + 8 * (r >> 1);
          if constexpr (PC == 128) {
            const uint4 v = lds128(vt + p * (16 * PC) + at_offset<PC>(token, g));
            vw[r][0] = v.x;
            vw[r][1] = v.y;
            vw[r][2] = v.z;
            vw[r][3] = v.w;
          } else {
            const uint2 v = lds64(vt + at_offset<PC>(token, g >> 1) + (g & 1) * 8);
            vw[r][0] = v.x;
            vw[r][1] = v.y;
          }
          if (tail && (wrong || (t << 4) + token >= see_last)) {  // 0 times what lies there may be NaN
#pragma unroll
            for (int i = 0; i < PC / 32; ++i) vw[r][i] = 0u;
          }
        }
        if (masked && !wrong) {
          // Tokens that only some queries of the group see: a NaN among their values belongs to
          // those alone, so it leaves the product below and is added where it is seen.
          uint32_t found = 0u;
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int i = 0; i < PC / 32; ++i) found |= __vcmpeq4(vw[r][i] & 0x7f7f7f7fu, 0x7f7f7f7fu);
          if (__any_sync(0xffffffffu, found != 0u)) {
            uint32_t see[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const int token = (t << 4) + 8 * (q >> 1) + 2 * c;
              see[q] = (token < limit[q & 1] ? 0x3c00u : 0u) | (token + 1 < limit[q & 1] ? 0x3c000000u : 0u);
            }
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
              for (int q = 0; q < 4; ++q) {
                const uint32_t pick = (uint32_t)(q | ((q + 4) << 4));
                float count[4] = {};
                mma_f16(count, see, f16_of_e4m3(__byte_perm(one[0], one[1], pick)), f16_of_e4m3(__byte_perm(one[2], one[3], pick)));
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (count[e] > 0.0f) o[p * NB + 4 * i + q][e] = __int_as_float(0x7fffffff);
              }
            }
          }
        }
#pragma unroll
        for (int i = 0; i < PC / 32; ++i) {
          const uint32_t t0 = __byte_perm(vw[0][i], vw[1][i], 0x5140), t1 = __byte_perm(vw[2][i], vw[3][i], 0x5140);
          const uint32_t u0b = __byte_perm(vw[0][i], vw[1][i], 0x7362), u1b = __byte_perm(vw[2][i], vw[3][i], 0x7362);
          mma_f16(o[p * NB + 4 * i], pa, f16_of_e4m3(t0), f16_of_e4m3(t1));
          mma_f16(o[p * NB + 4 * i + 1], pa, f16_of_e4m3(t0 >> 16), f16_of_e4m3(t1 >> 16));
          mma_f16(o[p * NB + 4 * i + 2], pa, f16_of_e4m3(u0b), f16_of_e4m3(u1b));
          mma_f16(o[p * NB + 4 * i + 3], pa, f16_of_e4m3(u0b >> 16), f16_of_e4m3(u1b >> 16));
        }
      }
      __syncwarp();
    }
    asm volatile("cp.async.wait_all;" ::: "memory");

#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    }
    // Lane (g, c) holds columns c * PC / 4 .. of rows g and g + 8: o[p * NB + i][2h + e] is column
    // p * PC + c * PC / 4 + e * NB + i.
    if (tile0 == 0 && tile1 == rw.nt) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (g + 8 * h < rows_here) {
          const int rr = mt * 16 + g + 8 * h, qi = rr / a.per, qh = head * a.per + rr - qi * a.per;
          const float f = l[h] == 0.0f ? 0.0f : ex2(w[h] - AT_BIAS - m[h]) / l[h];
          uint16_t* dst = reinterpret_cast<uint16_t*>(a.out) + (int64_t)(start + qi) * a.o_st + (int64_t)qh * a.o_sh;
#pragma unroll
          for (int p = 0; p < NP; ++p)
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
              for (int i = 0; i < NB; i += 8) {
                uint32_t pk[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                  float x0 = o[p * NB + i + 2 * q][2 * h + e] * f, x1 = o[p * NB + i + 2 * q + 1][2 * h + e] * f;
                  if (l[h] == 0.0f) x0 = x1 = 0.0f;
                  if (DT == LSS_DTYPE_BF16) {
                    const __nv_bfloat162 v = __floats2bfloat162_rn(x0, x1);
                    pk[q] = *reinterpret_cast<const uint32_t*>(&v);
                  } else {
                    const __half2 v = __floats2half2_rn(x0, x1);
                    pk[q] = *reinterpret_cast<const uint32_t*>(&v);
                  }
                }
                uint16_t* d = dst + p * PC + c * (PC / 4) + e * NB + i;
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
          if (a.lse && c == 0)
            a.lse[(int64_t)(start + qi) * (a.heads * a.per) + qh] = l[h] == 0.0f ? -INFINITY : (m[h] + log2f(l[h])) * LN2;
        }
      }
    } else {
      float* dst = a.part + (worker * 2 + (tile0 == 0 ? 1 : 0)) * (48 + 16 * D);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int rr = g + 8 * h;
        if (rr < rows_here) {
          if (c == 0) {
            dst[rr] = m[h];
            dst[16 + rr] = l[h];
            dst[32 + rr] = w[h];
          }
#pragma unroll
          for (int p = 0; p < NP; ++p)
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
              for (int i = 0; i < NB; i += 4) {
                float4 v;
                v.x = o[p * NB + i][2 * h + e];
                v.y = o[p * NB + i + 1][2 * h + e];
                v.z = o[p * NB + i + 2][2 * h + e];
                v.w = o[p * NB + i + 3][2 * h + e];
                *reinterpret_cast<float4*>(dst + 48 + rr * D + p * PC + c * (PC / 4) + e * NB + i) = v;
              }
        }
      }
      if (tile0 > 0) {  // the first cut inside its group joins the pieces
        const int64_t from = pos - tile0;
        const bool owner = from >= (worker - 1) * each;
        const int pieces = owner ? (int)((from + rw.nt - 1) / each - worker + 2) : 0;
        if (lane == 0) a.meta[worker] = make_int4(row, item, pieces, 0);
        wrote_meta = true;
      }
    }
    pos += tile1 - tile0;
    if (pos < end && pos - excl >= (int64_t)a.heads * rw.mt * rw.nt) {
      excl += (int64_t)a.heads * rw.mt * rw.nt;
      do ++row; while (row < a.B - 1 && at_row(a, row).n == 0);
    }
  }
  if (!wrote_meta && lane == 0) a.meta[worker] = make_int4(0, 0, 0, 0);
}

// Adds up the pieces of the groups that were cut: one CTA per worker, most with nothing to do.
template <int D, int DT>
__global__ void __launch_bounds__(256) lss_attend_join_kernel(AttendArgs a) {
  pdl_wait();
  const int64_t worker = blockIdx.x;
  const int4 me = a.meta[worker];
  if (me.z == 0) return;
  const AtRow rw = at_row(a, me.x);
  const int head = me.y / rw.mt, mt = me.y - head * rw.mt;
  const int rows_here = min(16, rw.n * a.per - mt * 16);
  constexpr int64_t PS = 48 + 16 * D;
  // Piece 0 is the last one of the worker before, the others the first ones of their workers.
  const float* p0 = a.part + ((worker - 1) * 2 + 1) * PS;
  const float* p1 = a.part + worker * 2 * PS;
  for (int x = threadIdx.x; x < rows_here * (D / 4); x += 256) {
    const int rr = x / (D / 4), d = (x % (D / 4)) * 4;
    float m = p0[rr], w = p0[32 + rr];
    for (int i = 0; i < me.z - 1; ++i) {
      m = fmaxf(m, p1[i * 2 * PS + rr]);
      w = fmaxf(w, p1[i * 2 * PS + 32 + rr]);
    }
    const float mu = m == -INFINITY ? 0.0f : m, wu = w == -INFINITY ? 0.0f : w;
    float l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int i = -1; i < me.z - 1; ++i) {
      const float* p = i < 0 ? p0 : p1 + i * 2 * PS;
      l += p[16 + rr] * ex2(p[rr] - mu);
      const float f = ex2(p[32 + rr] - wu);
      const float4 v = *reinterpret_cast<const float4*>(p + 48 + rr * D + d);
      o.x += v.x * f;
      o.y += v.y * f;
      o.z += v.z * f;
      o.w += v.w * f;
    }
    const float f = l == 0.0f ? 0.0f : ex2(w - AT_BIAS - m) / l;
    if (l == 0.0f) o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const int r2 = mt * 16 + rr, qi = r2 / a.per, qh = head * a.per + r2 - qi * a.per;
    const int64_t tok = a.starts[me.x] + qi;
    uint16_t* dst = reinterpret_cast<uint16_t*>(a.out) + tok * a.o_st + (int64_t)qh * a.o_sh + d;
    const float y[4] = {o.x * f, o.y * f, o.z * f, o.w * f};
#pragma unroll
    for (int q = 0; q < 4; ++q)
      dst[q] = DT == LSS_DTYPE_BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(y[q])) : __half_as_ushort(__float2half_rn(y[q]));
    if (a.lse && d == 0) a.lse[tok * (a.heads * a.per) + qh] = l == 0.0f ? -INFINITY : (m + log2f(l)) * LN2;
  }
}

}  // namespace lss
