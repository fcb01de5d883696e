// lss_attend_tc.cuh — the attention of lss_attend.cuh for prompt chunks: many query rows per key head,
// on the fifth-generation tensor cores (tcgen05, sums in tensor memory).
#pragma once

#include <type_traits>

#include "lss_attend.cuh"
#include "lss_int4_tc.cuh"

namespace lss {

constexpr int PA_ROWS = 256;   // query rows of a group: two tiles of 128
constexpr int PA_KT = 128;     // tokens of a tile of keys and values
constexpr int PA_HT = 64;      // tokens that a softmax step takes: half a tile
constexpr int PA_CONV = 7;     // warps that widen keys and values (16 in all: 128 registers a thread)
constexpr int PA_NT = (8 + PA_CONV + 1) * 32;

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

// Tiles of tokens that the last query of a group sees; units of a row.
__device__ __forceinline__ int pa_tiles(const AttendArgs& a, const AtRow& w, int mt) {
  const int last = min((mt + 1) * PA_ROWS, w.n * a.per) - 1;
  return (w.len - w.n + last / a.per + 1 + PA_KT - 1) / PA_KT;
}
__device__ __noinline__ int64_t pa_units(const AttendArgs& a, int r) {
  const AtRow w = at_row<PA_ROWS / 8>(a, r);
  int64_t n = 0;
  for (int mt = 0; mt < w.mt; ++mt) n += pa_tiles(a, w, mt);
  return n * a.heads;
}
// (token, head) of a query row and of the ones that follow it.
struct PaRows {
  int qi, h;
  __device__ __forceinline__ PaRows(const AttendArgs& a, int row) : qi(row / a.per), h(row - row / a.per * a.per) {}
  __device__ __forceinline__ void next(const AttendArgs& a, int rows) {
    h += rows;
    while (h >= a.per) {
      h -= a.per;
      ++qi;
    }
  }
};
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

// Where 16 bytes (8 values) `q` of row `r` lie in an operand of 128 rows: panels of 64 columns, a
// 128-byte line per row, pieces permuted by the row (the 128-byte swizzle).
__device__ __forceinline__ uint32_t pa_place(int r, int q) {
  return (uint32_t)((q >> 3) * (128 * 128) + r * 128 + (((q & 7) ^ (r & 7)) << 4));
}

// o = softmax(c q K^T) V for groups of 256 query rows (`per` heads times new tokens of one row and key head).
//
// Two tiles of 128 rows have a warpgroup each, a thread per row, and take 64 tokens a step: while it takes the
// softmax of a step's scores, the next step's are under way.  Scores S = Q K^T (two places of 128 x 64, f32) lie in
// tensor memory, the weights take their place as f16, the sums O stay there for the whole group.  Keys and
// values come as e4m3 and are widened to f16 by seven warps into two stages of shared memory, once for
// 256 rows (exact; 16 rows at a time, the widening is what bounds lss_attend_kernel here).
// Scales and the power of two of a query row act as in lss_attend_kernel; the weight of V is
// p 2^(m + log2(v scale) - W + 10) from the softmax's own p, one exponential per score.  Both running
// maxima may lag by 2^5, so that O is rarely rescaled.
// NaN among the values is kept out of the products (0 NaN of a masked place would spoil the row) and
// held as the first position per column from which it is seen.
// The units (group, tile of 128 tokens that it sees) are cut into equal ranges, one per CTA; pieces of a
// group are added up by lss_attend_tc_join_kernel.
// Measured: 296 to 416 new tokens over 3,000 to 5,300 (four rows, 32 query, 8 key heads of 128) 222 to 240 us, 410 to 450
// TFLOP/s, against 640 us with lss_attend_kernel; D = 64 165 to 185 us.  About 5,000 cycles per 256 x 128 scores at 48 % issue: waits for
// tensor memory and barriers between steps are what is left above the bounds.
// Bound by the exponentials (16 per cycle and SM: 2048 cycles per 256 x 128 scores) and the tensor pipe (the same
// number of cycles at D = 128).
template <int D, int DT>
__global__ void __launch_bounds__(PA_NT, 1) lss_attend_tc_kernel(AttendArgs a) {
  constexpr int CH = D / 8;                // 16-byte pieces of a row in f16
  constexpr int OPB = 128 * D * 2;         // bytes of a 128-row operand
  constexpr int PIECES = PA_KT * D / 16;   // 16-byte pieces of a tile in e4m3
  constexpr int PER_T = (PIECES + PA_CONV * 32 - 1) / (PA_CONV * 32);
  constexpr uint32_t NOWHERE = 0x7fffffff;
  extern __shared__ __align__(1024) unsigned char pa_dyn[];
  __shared__ __align__(8) uint64_t kfull[2], kempty[2], vfull[2], vempty[2], sfull[2][2], pready[2][2], pvdone[2], ofull[2], qready;
  __shared__ uint32_t tmem_base;
  __shared__ int failed;
  __shared__ float2 sscale[4][8];          // scales of the tile's 16-token parts: of K (< 0: not seen), log2 of that of V
  __shared__ int nan_from[D];              // first position with a NaN among the values of a column
  __shared__ int64_t scr[PA_NT / 32], found_lo;
  __shared__ int found, any_nan;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  unsigned char* base = pa_dyn + ((1024 - (saddr(pa_dyn) & 1023)) & 1023);
  unsigned char* qs = base;                // two query operands
  unsigned char* ksm = base + 2 * OPB;     // two stages of keys
  unsigned char* vsm = base + 4 * OPB;     // two stages of values

  if (warp == 0) tc_alloc(&tmem_base, 512);
  if (tid == 0) {
    failed = 0;
    for (int i = 0; i < 2; ++i) {
      mbar_init(&kfull[i], PA_CONV);
      mbar_init(&vfull[i], PA_CONV);
      mbar_init(&kempty[i], 1);
      mbar_init(&vempty[i], 1);
      for (int h = 0; h < 2; ++h) {
        mbar_init(&sfull[i][h], 1);
        mbar_init(&pready[i][h], 4);
      }
      mbar_init(&pvdone[i], 1);
      mbar_init(&ofull[i], 1);
    }
    mbar_init(&qready, 8);
    fence_barrier_init();
  }
  tc_before_sync();
  __syncthreads();
  tc_after_sync();
  const uint32_t tmem = tmem_base;
  const uint32_t s_at[2] = {tmem, tmem + 128}, o_at[2] = {tmem + 256, tmem + 256 + 128};

  // ---- the CTA's range of units (group of query rows, tile of tokens)
  int64_t total = 0;
  for (int r = tid; r < a.B; r += PA_NT) total += pa_units(a, r);
  total = pa_sum(total, scr);
  const int64_t each = max((total + gridDim.x - 1) / (int64_t)gridDim.x, (int64_t)1);
  int64_t pos = blockIdx.x * each;
  const int64_t end = min(pos + each, total);
  int4 join = make_int4(0, 0, 0, 0);

  uint32_t tiles = 0;       // K/V tiles of earlier groups
  uint32_t phases = 0;      // of the score barriers (softmax) or the weight barriers (products): bit 2 q + half
  uint32_t steps = 0, groups = 0;  // steps: of this warpgroup's query tile
  int row = -1, head = 0, mt = 0, tile0 = 0;
  if (pos < end) {  // where it begins: rows' units counted up by all threads
    int64_t before = 0;
    for (int r0 = 0; r0 < a.B && row < 0; r0 += PA_NT) {
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
      row = found;
    }
    const AtRow rw = at_row<PA_ROWS / 8>(a, row);
    const int64_t per_head = pa_units(a, row) / a.heads, rel = pos - found_lo;
    head = (int)(rel / per_head);
    int64_t u = rel - head * per_head;
    mt = rw.mt - 1;  // later groups see more: they come first
    while (u >= pa_tiles(a, rw, mt)) u -= pa_tiles(a, rw, mt--);
    tile0 = (int)u;
  }
  while (pos < end) {
    const AtRow rw = at_row<PA_ROWS / 8>(a, row);
    const int start = a.starts[row], ctx = rw.len - rw.n;
    const int rows_here = min(PA_ROWS, rw.n * a.per - mt * PA_ROWS);
    const int nq = rows_here > 128 ? 2 : 1;
    const int see_last = ctx + (mt * PA_ROWS + rows_here - 1) / a.per + 1;
    const int nt = pa_tiles(a, rw, mt), tile1 = (int)min((int64_t)nt, tile0 + (end - pos));
    const bool whole = tile0 == 0 && tile1 == nt;
    const int i0 = tile0 * 2, i1 = min(tile1 * 2, (see_last + PA_HT - 1) / PA_HT);  // steps of 64 tokens
    float* piece = a.part + ((size_t)blockIdx.x * 2 + (tile0 == 0 ? 1 : 0)) * pa_piece(D);
    for (int i = tid; i < D; i += PA_NT) nan_from[i] = NOWHERE;
    if (tid == 0) any_nan = 0;
    __syncthreads();  // and nobody reads the last group's any more

    if (warp < 8) {
      // ---- a thread per query row
      const int q = warp >> 2, r = (warp & 3) * 32 + lane, rr = q * 128 + r;
      const bool in = rr < rows_here;
      const int qi = in ? (mt * PA_ROWS + rr) / a.per : 0;
      const int qh = head * a.per + (in ? mt * PA_ROWS + rr - qi * a.per : 0);
      const int limit = in ? ctx + qi + 1 : 0;
      const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
      float fq = fabsf(a.scale);
      // Loops of this part, and of the one behind the tiles, stay rolled: code that runs once per group comes from
      // the L2 cache instruction line by instruction line (unrolled, they took 15 us per group).
      if (q < nq) {
        unsigned char* mine = qs + q * OPB;
        // The warp's 32 rows, CH lanes each, as they are.
        PaRows walk(a, mt * PA_ROWS + q * 128 + (warp & 3) * 32 + lane / CH);
#pragma unroll 1
        for (int i = 0; i < CH; ++i) {
          const int r2 = (warp & 3) * 32 + (i * 32 + lane) / CH;
          const bool in2 = q * 128 + r2 < rows_here;
          const uint16_t* src = reinterpret_cast<const uint16_t*>(a.q) +
                                (in2 ? (int64_t)(start + walk.qi) * a.q_st + (int64_t)(head * a.per + walk.h) * a.q_sh + (lane % CH) * 8 : 0);
          unsigned char* to = mine + pa_place(r2, lane % CH);
          if (a.aligned) {
            cp_async16z(saddr(to), src, in2 ? 16 : 0);
          } else {
            uint32_t u[4] = {0, 0, 0, 0};
            if (in2) {
#pragma unroll
              for (int e = 0; e < 4; ++e) u[e] = (uint32_t)src[2 * e] | ((uint32_t)src[2 * e + 1] << 16);
            }
            *reinterpret_cast<uint4*>(to) = make_uint4(u[0], u[1], u[2], u[3]);
          }
          walk.next(a, 32 / CH);
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncwarp();
        // bf16 to f16, a thread per row: largest exponent to 0, the power of two goes into the row's factor.
        float down = 1.0f;
        if (DT == LSS_DTYPE_BF16) {
          uint32_t top = 0;  // magnitudes of bf16 order as whole numbers do
#pragma unroll 4
          for (int i = 0; i < CH; ++i) {
            const uint4 v = *reinterpret_cast<const uint4*>(mine + pa_place(r, i));
            top = __vmaxu2(__vmaxu2(top, v.x & 0x7fff7fffu), __vmaxu2(v.y & 0x7fff7fffu, __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu)));
          }
          top = max(top & 0xffffu, top >> 16);
          const int e = min(max((int)(top >> 7) - 127, -126), 126);
          down = __uint_as_float((uint32_t)(127 - e) << 23);
          fq *= __uint_as_float((uint32_t)(127 + e) << 23);
        }
        const uint32_t sign = a.scale < 0.0f ? 0x80008000u : 0u;  // scores are compared before they are scaled
        if (DT == LSS_DTYPE_BF16 || sign != 0u) {
#pragma unroll 2
          for (int i = 0; i < CH; ++i) {
            uint4* at = reinterpret_cast<uint4*>(mine + pa_place(r, i));
            const uint4 v = *at;
            uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if (DT == LSS_DTYPE_BF16) {
                const __half2 h = __floats2half2_rn(__uint_as_float(u[e] << 16) * down, __uint_as_float(u[e] & 0xffff0000u) * down);
                u[e] = *reinterpret_cast<const uint32_t*>(&h);
              }
              u[e] ^= sign;
            }
            *at = make_uint4(u[0], u[1], u[2], u[3]);
          }
        }
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive_local(&qready);

      float m = -INFINITY, l = 0.0f, w = -INFINITY;
      if (q < nq) {
        // The first row of the warp sees least.
        const int see_warp = ctx + (mt * PA_ROWS + q * 128 + (warp & 3) * 32) / a.per + 1;
        for (int i = i0; i < i1; ++i, ++steps) {
          const int half = i & 1, at = i * PA_HT;
          tc_wait(&sfull[q][half], (phases >> half) & 1, &failed);
          phases ^= 1u << half;
          tc_after_sync();
          const uint32_t s_here = s_at[q] + lanes + 64 * half;
          const float2* sc = &sscale[(tiles + (i >> 1) - tile0) & 3][4 * half];
          bool masked = at + PA_HT > see_warp;
#pragma unroll
          for (int g = 0; g < 4; ++g) masked |= sc[g].x < 0.0f;
          uint32_t x[4][16];
#pragma unroll
          for (int g = 0; g < 4; ++g) tc_ld16(s_here + 16 * g, x[g]);
          tc_wait_ld();
          // Largest score, and largest weight of V.
          float top = -INFINITY, topw = -INFINITY, least = INFINITY;
          auto maxima = [&](auto mask_c) {
            constexpr bool with_mask = decltype(mask_c)::value;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const float2 k = sc[g];
              float t = -INFINITY;
#pragma unroll
              for (int e = 0; e < 16; ++e)
                if (!with_mask || at + 16 * g + e < limit) t = fmaxf(t, __uint_as_float(x[g][e]));
              if (with_mask && (k.x < 0.0f || at + 16 * g >= limit)) continue;
              t = fmaxf(t * (fq * k.x), -FLT_MAX);  // -inf and NaN: seen, unlike what leaves m at -inf
              top = fmaxf(top, t);
              topw = fmaxf(topw, t + k.y);
              least = fminf(least, k.y);
            }
          };
          if (masked) maxima(std::true_type{}); else maxima(std::false_type{});
          if (__any_sync(0xffffffffu, top > m + AT_SLACK || topw > w + AT_SLACK)) {
            const float mn = fmaxf(m, top), wn = fmaxf(w, topw);
            l *= ex2(m - (mn == -INFINITY ? 0.0f : mn));
            const float shrink = ex2(w - (wn == -INFINITY ? 0.0f : wn));
            m = mn;
            w = wn;
            if (i > i0) {  // the sums so far, once the products of the step before are in them
              tc_wait(&pvdone[q], (steps - 1) & 1, &failed);
              tc_after_sync();
#pragma unroll 1
              for (int d = 0; d < D; d += 16) {
                uint32_t x[16];
                tc_ld16(o_at[q] + lanes + d, x);
                tc_wait_ld();
#pragma unroll
                for (int e = 0; e < 16; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) * shrink);
                tc_st16(o_at[q] + lanes + d, x);
              }
            }
          }
          const float mu = m == -INFINITY ? 0.0f : m, wu = w == -INFINITY ? 0.0f : w;
          // A token's weight of V is 2^z, z = s + log2(v scale) - W + 10; its share p = 2^(s - m) of the softmax
          // differs by a factor of its part, so that one exponential does for both: p = 2^z 2^(-shift).  Where the factor
          // is far from 1 (a block of zeros has the scale 2^-126) p would be lost: then p itself is taken.
          const bool apart = __any_sync(0xffffffffu, mu + least - wu + AT_BIAS < -60.0f);
          auto weights = [&](auto mask_c, auto share_c) {
            constexpr bool with_mask = decltype(mask_c)::value, by_share = decltype(share_c)::value;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const float2 k = sc[g];
              const float fg = fq * k.x, shift = fminf(mu + k.y - wu + AT_BIAS, 126.0f);
              const float add = by_share ? -mu : k.y - wu + AT_BIAS, gain = by_share ? ex2(shift) : 0.0f;
              uint32_t p[8];
              float part = 0.0f;
#pragma unroll
              for (int e = 0; e < 16; e += 2) {
                float y0 = fmaf(__uint_as_float(x[g][e]), fg, add), y1 = fmaf(__uint_as_float(x[g][e + 1]), fg, add);
                if (with_mask) {
                  if (k.x < 0.0f || at + 16 * g + e >= limit) y0 = -INFINITY;
                  if (k.x < 0.0f || at + 16 * g + e + 1 >= limit) y1 = -INFINITY;
                }
                float p0 = ex2(y0), p1 = ex2(y1);
                part += p0 + p1;
                if (by_share) {
                  p0 *= gain;
                  p1 *= gain;
                }
                const __half2 v = __floats2half2_rn(p0, p1);
                p[e / 2] = *reinterpret_cast<const uint32_t*>(&v);
              }
              if (by_share) l += part;
              else if (!with_mask || part != 0.0f) l = fmaf(part, ex2(-shift), l);
              tc_st8(s_here + 8 * g, p);  // over scores that have been read
            }
          };
          if (masked) weights(std::true_type{}, std::true_type{});
          else if (apart) weights(std::false_type{}, std::true_type{});
          else weights(std::false_type{}, std::false_type{});
          tc_wait_st();
          tc_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive_local(&pready[q][half]);
        }
        tc_wait(&ofull[q], groups & 1, &failed);
        tc_after_sync();
        if (!whole && rr < rows_here) {  // a piece: its state as it is
          piece[rr] = m;
          piece[PA_ROWS + rr] = l;
          piece[2 * PA_ROWS + rr] = w;
        }
        const bool none = m == -INFINITY, bad = *(volatile int*)&failed, spoiled = bad || any_nan;
        const AtFactor fin(m, l, w);
#pragma unroll 1
        for (int i = 0; i < D; i += 16) {
          uint32_t x[16];
          tc_ld16(o_at[q] + lanes + i, x);
          tc_wait_ld();
          if (!whole) {
            float* to = piece + 3 * PA_ROWS + rr * D + i;
            if (in)
#pragma unroll
              for (int e = 0; e < 16; e += 4)
                *reinterpret_cast<uint4*>(to + e) = bad ? make_uint4(NOWHERE, NOWHERE, NOWHERE, NOWHERE) : make_uint4(x[e], x[e + 1], x[e + 2], x[e + 3]);
          } else {
            uint32_t pk[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              float y[2];
#pragma unroll
              for (int z = 0; z < 2; ++z) {
                y[z] = none ? 0.0f : fin(__uint_as_float(x[2 * e + z]));
                if (spoiled && (bad || nan_from[i + 2 * e + z] < limit)) y[z] = __int_as_float(0x7fffffff);
              }
              pk[e] = at_pack<DT>(y[0], y[1]);
            }
            // Into the place of the queries, which no product reads any more.
            *reinterpret_cast<uint4*>(qs + q * OPB + pa_place(r, i / 8)) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
            *reinterpret_cast<uint4*>(qs + q * OPB + pa_place(r, i / 8 + 1)) = make_uint4(pk[4], pk[5], pk[6], pk[7]);
          }
        }
        if (whole) {
          __syncwarp();
          PaRows walk(a, mt * PA_ROWS + q * 128 + (warp & 3) * 32 + lane / CH);
#pragma unroll 1
          for (int i = 0; i < CH; ++i) {
            const int r2 = (warp & 3) * 32 + (i * 32 + lane) / CH;
            if (q * 128 + r2 < rows_here) {
              uint16_t* out = reinterpret_cast<uint16_t*>(a.out) + (int64_t)(start + walk.qi) * a.o_st + (int64_t)(head * a.per + walk.h) * a.o_sh + (lane % CH) * 8;
              const uint4 v = *reinterpret_cast<const uint4*>(qs + q * OPB + pa_place(r2, lane % CH));
              if (a.aligned) {
                *reinterpret_cast<uint4*>(out) = v;
              } else {
                const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  out[2 * e] = (uint16_t)u[e];
                  out[2 * e + 1] = (uint16_t)(u[e] >> 16);
                }
              }
            }
            walk.next(a, 32 / CH);
          }
        }
        if (in && whole && a.lse) a.lse[(int64_t)(start + qi) * (a.heads * a.per) + qh] = none ? -INFINITY : (m + log2f(l)) * LN2;
        tc_before_sync();
      }
    } else if (warp < 8 + PA_CONV) {
      // ---- widens keys and values, a tile ahead of the products
      const int ct = tid - 256;
      const int32_t* trow = a.table + row * a.table_stride;
      const int bsm = (1 << a.bs_shift) - 1;
      uint4 kr[PER_T], vr[PER_T];
      int ids[PER_T], ids_next[PER_T], part_id = -1, part_next = -1;
      float ksn = 0.0f, lvn = 0.0f;
      // Block ids of the thread's pieces of tile j (-1: not seen), a tile ahead of their use; then keys with the
      // scales, and values, each as soon as the registers of the tile before are free.
      auto locate = [&](int j) {
        auto id = [&](int t) {
          const int page = t < see_last && j < tile1 ? __ldg(trow + (t >> a.bs_shift)) : -1;
          return (unsigned)page < (unsigned)a.num_blocks ? page : -1;
        };
#pragma unroll
        for (int i = 0; i < PER_T; ++i) {
          const int p = ct + i * PA_CONV * 32;
          ids_next[i] = p < PIECES ? id(j * PA_KT + p / (D / 16)) : -1;
        }
        if (ct < 8) part_next = id(j * PA_KT + ct * 16);
      };
      auto advance = [&]() {
#pragma unroll
        for (int i = 0; i < PER_T; ++i) ids[i] = ids_next[i];
        part_id = part_next;
      };
      auto fetch = [&](const uint8_t* from, uint4 (&to)[PER_T], int j) {
#pragma unroll
        for (int i = 0; i < PER_T; ++i) {
          const int p = ct + i * PA_CONV * 32, t = j * PA_KT + p / (D / 16), cc = p % (D / 16);
          to[i] = ids[i] >= 0 ? __ldg(reinterpret_cast<const uint4*>(from + (((int64_t)ids[i] * a.heads + head) << a.bs_shift) * D + (t & bsm) * D + cc * 16))
                              : make_uint4(0, 0, 0, 0);
        }
      };
      auto fetch_scales = [&]() {
        if (ct < 8) {
          ksn = part_id >= 0 ? __ldg(a.ks + (int64_t)part_id * a.heads + head) : -1.0f;
          lvn = part_id >= 0 ? lg2(__ldg(a.vs + (int64_t)part_id * a.heads + head)) : -INFINITY;
        }
      };
      auto widen = [&](const uint4& v, unsigned char* to, int t, int cc) {
        const uint32_t u[4] = {v.x, v.y, v.z, v.w};
        const uint4 lo = make_uint4(f16_of_e4m3(u[0]), f16_of_e4m3(u[0] >> 16), f16_of_e4m3(u[1]), f16_of_e4m3(u[1] >> 16));
        const uint4 hi = make_uint4(f16_of_e4m3(u[2]), f16_of_e4m3(u[2] >> 16), f16_of_e4m3(u[3]), f16_of_e4m3(u[3] >> 16));
        // Lanes of the second panel store their second piece first: 8 lanes, 8 bank groups.
        const bool swap = D > 64 && cc >= 4;
        *reinterpret_cast<uint4*>(to + pa_place(t, 2 * cc + swap)) = swap ? hi : lo;
        *reinterpret_cast<uint4*>(to + pa_place(t, 2 * cc + !swap)) = swap ? lo : hi;
      };
      locate(tile0);
      advance();
      locate(tile0 + 1);
      fetch(a.kc, kr, tile0);
      fetch_scales();
      fetch(a.vc, vr, tile0);
      for (int j = tile0; j < tile1; ++j) {
        const uint32_t n = tiles + j - tile0, st = n & 1;
        if (n >= 2) tc_wait(&kempty[st], ((n >> 1) - 1) & 1, &failed);
#pragma unroll
        for (int i = 0; i < PER_T; ++i) {
          const int p = ct + i * PA_CONV * 32;
          if (p < PIECES) widen(kr[i], ksm + st * OPB, p / (D / 16), p % (D / 16));
        }
        if (ct < 8) {
          sscale[n & 3][ct] = make_float2(ksn, lvn);
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive_local(&kfull[st]);
        advance();
        if (j + 1 < tile1) {
          fetch(a.kc, kr, j + 1);
          fetch_scales();
          locate(j + 2);
        }
        if (n >= 2) tc_wait(&vempty[st], ((n >> 1) - 1) & 1, &failed);
#pragma unroll
        for (int i = 0; i < PER_T; ++i) {
          const int p = ct + i * PA_CONV * 32, t = p / (D / 16), cc = p % (D / 16);
          uint32_t u[4] = {vr[i].x, vr[i].y, vr[i].z, vr[i].w};
          uint32_t any = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) any |= (u[e] & 0x7f7f7f7fu) + 0x01010101u;  // a byte of 0x7f carries into its sign
          if (any & 0x80808080u) {
            any_nan = 1;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t nan = __vcmpeq4(u[e] & 0x7f7f7f7fu, 0x7f7f7f7fu);
              for (int z = 0; z < 4; ++z)
                if ((nan >> (8 * z)) & 1u) atomicMin(&nan_from[cc * 16 + 4 * e + z], j * PA_KT + t);
              u[e] &= ~nan;
            }
          }
          if (p < PIECES) widen(make_uint4(u[0], u[1], u[2], u[3]), vsm + st * OPB, t, cc);
        }
        if (j + 1 < tile1) fetch(a.vc, vr, j + 1);
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive_local(&vfull[st]);
      }
    } else {
      // ---- issues the products: scores of tile j follow the weighted values of tile j - 1, query tiles in turn
      constexpr uint32_t is = tc_idesc(false, PA_HT), io = tc_idesc(false, D) | (1u << 16);  // values: columns lie together
      tc_wait(&qready, groups & 1, &failed);
      auto score = [&](int q, int i) {
        const uint32_t n = tiles + (i >> 1) - tile0, st = n & 1, half = i & 1;
        if (q == 0 && half == 0) tc_wait(&kfull[st], (n >> 1) & 1, &failed);
        tc_after_sync();
        __syncwarp();
        if (!tc_elect() || *(volatile int*)&failed) return;
        const uint32_t q0 = tc_desc_lo(saddr(qs + q * OPB)), k0 = tc_desc_lo(saddr(ksm + st * OPB) + half * (PA_HT * 128));
#pragma unroll
        for (int s = 0; s < D / 16; ++s) {
          const uint32_t off = (uint32_t)((s >> 2) * (128 * 128) + (s & 3) * 32) / 16;
          tc_mma_ss(s_at[q] + 64 * half, q0 + off, TC_DESC_HI, k0 + off, TC_DESC_HI, is, s > 0);
        }
        tc_commit(&sfull[q][half]);
        if (q == nq - 1 && (half == 1 || i == i1 - 1)) tc_commit(&kempty[st]);
      };
      auto weigh = [&](int q, int i) {
        const uint32_t n = tiles + (i >> 1) - tile0, st = n & 1, half = i & 1;
        tc_wait(&pready[q][half], (phases >> (2 * q + half)) & 1, &failed);
        phases ^= 1u << (2 * q + half);
        if (q == 0 && half == 0) tc_wait(&vfull[st], (n >> 1) & 1, &failed);
        tc_after_sync();
        __syncwarp();
        if (!tc_elect() || *(volatile int*)&failed) return;
        // panels of 64 columns are 16 KB apart, groups of 8 tokens 1 KB
        const uint32_t v0 = (((saddr(vsm + st * OPB) + half * (PA_HT * 128)) >> 4) & 0x3fffu) | ((128u * 128u >> 4) << 16);
#pragma unroll
        for (int s = 0; s < PA_HT / 16; ++s)
          tc_mma_ts(o_at[q], s_at[q] + 64 * half + 8 * s, v0 + s * (2048 / 16), TC_DESC_HI, io, i > i0 || s > 0);
        tc_commit(&pvdone[q]);
        if (q == nq - 1 && (half == 1 || i == i1 - 1)) tc_commit(&vempty[st]);
      };
      // Scores are two steps ahead of the weighted values: the next ones wait when a warpgroup has its weights.
      for (int i = i0; i < min(i0 + 2, i1); ++i)
        for (int q = 0; q < nq; ++q) score(q, i);
#pragma unroll 1
      for (int i = i0; i < i1; ++i) {
#pragma unroll 1
        for (int q = 0; q < nq; ++q) {
          weigh(q, i);
          __syncwarp();
          if (i == i1 - 1 && tc_elect()) tc_commit(&ofull[q]);
          if (i + 2 < i1) score(q, i + 2);
        }
      }
      __syncwarp();
      if (nq == 1 && tc_elect()) tc_commit(&ofull[1]);  // its phase goes with the groups
    }
    __syncwarp();
    __syncthreads();
    if (!whole)
      for (int i = tid; i < D; i += PA_NT) reinterpret_cast<int*>(piece + 3 * PA_ROWS + PA_ROWS * D)[i] = nan_from[i];
    if (tile0 > 0) {  // the first cut inside its group joins the pieces
      const int64_t from = pos - tile0;
      if (from >= ((int64_t)blockIdx.x - 1) * each) join = make_int4(row, mt * a.heads + head, (int)((from + nt - 1) / each) - (int)blockIdx.x + 2, 0);
    }
    tiles += tile1 - tile0;
    ++groups;
    pos += tile1 - tile0;
    tile0 = 0;
    if (pos < end && --mt < 0) {  // next group of the head, next head, next row with work
      if (++head == a.heads) {
        head = 0;
        do ++row; while (row < a.B - 1 && at_row<PA_ROWS / 8>(a, row).n == 0);
      }
      mt = at_row<PA_ROWS / 8>(a, row).mt - 1;
    }
    __syncthreads();  // the positions of NaN are out
  }
  if (tid == 0) a.meta[blockIdx.x] = join;
  tc_before_sync();
  __syncthreads();
  tc_after_sync();
  if (*(volatile int*)&failed) {  // products may still run: they get a quarter of a second
    const long long t0 = clock64();
    while (clock64() - t0 < T4_WAIT / 4) __nanosleep(1000);
    __syncthreads();
  }
  if (warp == 0) tc_free(tmem, 512);
}

// Adds up the pieces of a group that was cut, the last one of the CTA before and the first ones of this
// CTA and those after it; 32 rows per CTA.
template <int D, int DT>
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
