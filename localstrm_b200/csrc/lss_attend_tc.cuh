// lss_attend_tc.cuh — the attention of lss_attend.cuh for prompt chunks: many query rows per key head,
// on the fifth-generation tensor cores (tcgen05, sums in tensor memory).
#pragma once

#include <type_traits>

#include "lss_attend.cuh"
#include "lss_int4_tc.cuh"

namespace lss {

constexpr int PA_ROWS = 256;   // query rows of a group: two tiles of 128
constexpr int PA_KT = 128;     // tokens of a tile
constexpr int PA_CONV = 8;     // warps that widen keys and values
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

// Where 16 bytes (8 values) `q` of row `r` lie in an operand of 128 rows: panels of 64 columns, a
// 128-byte line per row, pieces permuted by the row (the 128-byte swizzle).
__device__ __forceinline__ uint32_t pa_place(int r, int q) {
  return (uint32_t)((q >> 3) * (128 * 128) + r * 128 + (((q & 7) ^ (r & 7)) << 4));
}

// o = softmax(c q K^T) V for groups of 256 query rows (`per` heads times new tokens of one row and key head).
//
// Two tiles of 128 rows take turns on the tensor cores: while one warpgroup (a thread per row) takes
// the softmax of its scores, the products of the other run.  Scores S = Q K^T (128 x 128, f32) lie in tensor
// memory, the weights take their place as f16, the sums O stay there for the whole group.  Keys and
// values come as e4m3 and are widened to f16 by eight warps into two stages of shared memory, once for
// 256 rows (exact; 16 rows at a time, the widening is what bounds lss_attend_kernel here).
// Scales and the power of two of a query row act as in lss_attend_kernel; the weight of V is
// p 2^(m + log2(v scale) - W + 10) from the softmax's own p, one exponential per score.  Both running
// maxima may lag by 2^5, so that O is rarely rescaled.
// NaN among the values is kept out of the products (0 NaN of a masked place would spoil the row) and
// held as the first position per column from which it is seen.
// Bound by the exponentials (16 per cycle and SM: 2048 cycles per 256 x 128 scores) and the tensor pipe (the same
// number of cycles at D = 128).
template <int D, int DT>
__global__ void __launch_bounds__(PA_NT, 1) lss_attend_tc_kernel(AttendArgs a) {
  constexpr int CH = D / 8;                // 16-byte pieces of a row in f16
  constexpr int OPB = 128 * D * 2;         // bytes of a 128-row operand
  constexpr int PIECES = PA_KT * D / 16;   // 16-byte pieces of a tile in e4m3
  constexpr int PER_T = PIECES / (PA_CONV * 32);
  constexpr uint32_t LIST = 0x7fffffff;
  extern __shared__ __align__(1024) unsigned char pa_dyn[];
  __shared__ __align__(8) uint64_t kfull[2], kempty[2], vfull[2], vempty[2], sfull[2], pready[2], ofull[2], qready;
  __shared__ uint32_t tmem_base;
  __shared__ int failed;
  __shared__ float2 sscale[4][8];          // scales of the tile's 16-token parts: of K (< 0: not seen), log2 of that of V
  __shared__ int nan_from[D];              // first position with a NaN among the values of a column
  __shared__ int scr[PA_NT / 32];
  __shared__ int4 found;
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
      mbar_init(&sfull[i], 1);
      mbar_init(&pready[i], 4);
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

  uint32_t tiles = 0;       // K/V tiles of earlier groups
  uint32_t scount[2] = {0, 0}, groups = 0;
  // Groups in rounds of the grid's size, every second round the other way round: later rows tend to have less.
  for (int round = 0;; ++round) {
    const int item0 = round * (int)gridDim.x + (round & 1 ? (int)(gridDim.x - 1 - blockIdx.x) : (int)blockIdx.x);
    // ---- which row, key head and group: rows' groups counted up by all threads
    int rest = item0, row = -1;
    for (int r0 = 0; r0 < a.B && row < 0; r0 += PA_NT) {
      const int r = r0 + tid;
      int n = 0;
      if (r < a.B) {
        const AtRow w = at_row<PA_ROWS / 8>(a, r);
        n = a.heads * w.mt;
      }
      int x = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      if (lane == 31) scr[warp] = x;
      if (tid == 0) found.x = -1;
      __syncthreads();
      int before = 0, tot = 0;
#pragma unroll
      for (int i = 0; i < PA_NT / 32; ++i) {
        if (i < warp) before += scr[i];
        tot += scr[i];
      }
      const int lo = before + x - n;
      if (rest >= lo && rest < lo + n) found = make_int4(r, rest - lo, 0, 0);
      __syncthreads();
      const int4 f = found;
      __syncthreads();
      if (f.x >= 0) {
        row = f.x;
        rest = f.y;
      } else {
        rest -= tot;
      }
    }
    if (row < 0) break;  // places of later rounds lie further behind
    const AtRow rw = at_row<PA_ROWS / 8>(a, row);
    // Later groups see more: they come first.
    const int head = rest % a.heads, mt = rw.mt - 1 - rest / a.heads;
    const int start = a.starts[row], ctx = rw.len - rw.n;
    const int rows_here = min(PA_ROWS, rw.n * a.per - mt * PA_ROWS);
    const int nq = rows_here > 128 ? 2 : 1;
    const int see_last = ctx + (mt * PA_ROWS + rows_here - 1) / a.per + 1;
    const int nt = (see_last + PA_KT - 1) / PA_KT;
    for (int i = tid; i < D; i += PA_NT) nan_from[i] = LIST;
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
      if (q < nq) {
        const uint16_t* src = reinterpret_cast<const uint16_t*>(a.q) + (in ? (int64_t)(start + qi) * a.q_st + (int64_t)qh * a.q_sh : 0);
        auto piece = [&](int i) {
          uint4 v = make_uint4(0, 0, 0, 0);
          if (in) {
            if (a.aligned) {
              v = __ldg(reinterpret_cast<const uint4*>(src + 8 * i));
            } else {
              uint32_t* u = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
              for (int e = 0; e < 4; ++e) u[e] = (uint32_t)src[8 * i + 2 * e] | ((uint32_t)src[8 * i + 2 * e + 1] << 16);
            }
          }
          return v;
        };
        float down = 1.0f;
        if (DT == LSS_DTYPE_BF16) {  // largest exponent to 0
          float amax = 0.0f;
#pragma unroll 4
          for (int i = 0; i < CH; ++i) {
            const uint4 v = piece(i);
            const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float x0 = fabsf(__uint_as_float(u[e] << 16)), x1 = fabsf(__uint_as_float(u[e] & 0xffff0000u));
              if (x0 <= FLT_MAX) amax = fmaxf(amax, x0);
              if (x1 <= FLT_MAX) amax = fmaxf(amax, x1);
            }
          }
          const int e = min(max((int)(__float_as_uint(amax) >> 23) - 127, -126), 126);
          down = __uint_as_float((uint32_t)(127 - e) << 23);
          fq *= __uint_as_float((uint32_t)(127 + e) << 23);
        }
        const uint32_t sign = a.scale < 0.0f ? 0x80008000u : 0u;  // scores are compared before they are scaled
#pragma unroll 4
        for (int i = 0; i < CH; ++i) {
          const uint4 v = piece(i);
          uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (DT == LSS_DTYPE_BF16) {
              const __half2 h = __floats2half2_rn(__uint_as_float(u[e] << 16) * down, __uint_as_float(u[e] & 0xffff0000u) * down);
              u[e] = *reinterpret_cast<const uint32_t*>(&h);
            }
            u[e] ^= sign;
          }
          *reinterpret_cast<uint4*>(qs + q * OPB + pa_place(r, i)) = make_uint4(u[0], u[1], u[2], u[3]);
        }
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive_local(&qready);

      float m = -INFINITY, l = 0.0f, w = -INFINITY;
      if (q < nq) {
        // The first row of the warp sees least.
        const int see_warp = ctx + (mt * PA_ROWS + q * 128 + (warp & 3) * 32) / a.per + 1;
        for (int j = 0; j < nt; ++j) {
          tc_wait(&sfull[q], scount[q] & 1, &failed);
          ++scount[q];
          tc_after_sync();
          const int slot = (int)((tiles + j) & 3), pos = j * PA_KT;
          const float2* sc = sscale[slot];
          bool masked = pos + PA_KT > see_warp;
#pragma unroll
          for (int g = 0; g < 8; ++g) masked |= sc[g].x < 0.0f;
          // Largest score, and largest weight of V.  Sixteen columns at a time, the next ones on their way.
          float top = -INFINITY, topw = -INFINITY, least = INFINITY;
          auto maxima = [&](auto mask_c) {
            constexpr bool with_mask = decltype(mask_c)::value;
            uint32_t x[2][16];
            tc_ld16(s_at[q] + lanes, x[0]);
#pragma unroll
            for (int g = 0; g < 8; ++g) {
              tc_wait_ld();
              if (g < 7) tc_ld16(s_at[q] + lanes + 16 * (g + 1), x[(g + 1) & 1]);
              const float2 k = sc[g];
              float t = -INFINITY;
#pragma unroll
              for (int e = 0; e < 16; ++e)
                if (!with_mask || pos + 16 * g + e < limit) t = fmaxf(t, __uint_as_float(x[g & 1][e]));
              if (with_mask && (k.x < 0.0f || t == -INFINITY)) continue;
              t *= fq * k.x;
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
            if (j > 0) {  // the sums so far: their products were issued before these scores'
#pragma unroll
              for (int i = 0; i < D; i += 16) {
                uint32_t x[16];
                tc_ld16(o_at[q] + lanes + i, x);
                tc_wait_ld();
#pragma unroll
                for (int e = 0; e < 16; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) * shrink);
                tc_st16(o_at[q] + lanes + i, x);
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
            uint32_t x[2][16];
            tc_ld16(s_at[q] + lanes, x[0]);
#pragma unroll
            for (int g = 0; g < 8; ++g) {
              tc_wait_ld();
              if (g < 7) tc_ld16(s_at[q] + lanes + 16 * (g + 1), x[(g + 1) & 1]);
              const float2 k = sc[g];
              const float fg = fq * k.x, shift = fminf(mu + k.y - wu + AT_BIAS, 126.0f);
              const float add = by_share ? -mu : k.y - wu + AT_BIAS, gain = by_share ? ex2(shift) : 0.0f;
              uint32_t p[8];
              float part = 0.0f;
#pragma unroll
              for (int e = 0; e < 16; e += 2) {
                float y0 = fmaf(__uint_as_float(x[g & 1][e]), fg, add), y1 = fmaf(__uint_as_float(x[g & 1][e + 1]), fg, add);
                if (with_mask) {
                  if (k.x < 0.0f || pos + 16 * g + e >= limit) y0 = -INFINITY;
                  if (k.x < 0.0f || pos + 16 * g + e + 1 >= limit) y1 = -INFINITY;
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
              tc_st8(s_at[q] + lanes + 8 * g, p);  // over scores that have been read
            }
          };
          if (masked) weights(std::true_type{}, std::true_type{});
          else if (apart) weights(std::false_type{}, std::true_type{});
          else weights(std::false_type{}, std::false_type{});
          tc_wait_st();
          tc_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive_local(&pready[q]);
        }
        tc_wait(&ofull[q], groups & 1, &failed);
        tc_after_sync();
        const bool none = l == 0.0f, bad = *(volatile int*)&failed;
        const float fin = ex2(w - AT_BIAS - m) / l;
        uint16_t* out = reinterpret_cast<uint16_t*>(a.out) + (in ? (int64_t)(start + qi) * a.o_st + (int64_t)qh * a.o_sh : 0);
#pragma unroll
        for (int i = 0; i < D; i += 16) {
          uint32_t x[16];
          tc_ld16(o_at[q] + lanes + i, x);
          tc_wait_ld();
          if (in) {
            uint32_t pk[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              float y[2];
#pragma unroll
              for (int z = 0; z < 2; ++z) {
                y[z] = none ? 0.0f : __uint_as_float(x[2 * e + z]) * fin;
                if (bad || nan_from[i + 2 * e + z] < limit) y[z] = __int_as_float(0x7fffffff);
              }
              pk[e] = at_pack<DT>(y[0], y[1]);
            }
            if (a.aligned) {
              *reinterpret_cast<uint4*>(out + i) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
              *reinterpret_cast<uint4*>(out + i + 8) = make_uint4(pk[4], pk[5], pk[6], pk[7]);
            } else {
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                out[i + 2 * e] = (uint16_t)pk[e];
                out[i + 2 * e + 1] = (uint16_t)(pk[e] >> 16);
              }
            }
          }
        }
        if (in && a.lse) a.lse[(int64_t)(start + qi) * (a.heads * a.per) + qh] = none ? -INFINITY : (m + log2f(l)) * LN2;
        tc_before_sync();
      }
    } else if (warp < 8 + PA_CONV) {
      // ---- widens keys and values, a tile ahead of the products
      const int ct = tid - 256;
      const int32_t* trow = a.table + row * a.table_stride;
      const int bsm = (1 << a.bs_shift) - 1;
      uint4 kr[PER_T], vr[PER_T];
      float ksn = 0.0f, lvn = 0.0f;
      auto fetch = [&](int j) {
#pragma unroll
        for (int i = 0; i < PER_T; ++i) {
          const int p = ct + i * PA_CONV * 32, t = j * PA_KT + p / (D / 16), cc = p % (D / 16);
          kr[i] = vr[i] = make_uint4(0, 0, 0, 0);
          if (t < see_last) {
            const int page = trow[t >> a.bs_shift];
            if ((unsigned)page < (unsigned)a.num_blocks) {
              const int64_t at = ((((int64_t)page * a.heads + head) << a.bs_shift) + (t & bsm)) * D + cc * 16;
              kr[i] = __ldg(reinterpret_cast<const uint4*>(a.kc + at));
              vr[i] = __ldg(reinterpret_cast<const uint4*>(a.vc + at));
            }
          }
        }
        if (ct < 8) {
          const int t = j * PA_KT + ct * 16;
          ksn = -1.0f;
          lvn = -INFINITY;
          if (t < see_last) {
            const int page = trow[t >> a.bs_shift];
            if ((unsigned)page < (unsigned)a.num_blocks) {
              ksn = __ldg(a.ks + (int64_t)page * a.heads + head);
              lvn = lg2(__ldg(a.vs + (int64_t)page * a.heads + head));
            }
          }
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
      fetch(0);
      for (int j = 0; j < nt; ++j) {
        const uint32_t n = tiles + j, st = n & 1;
        if (n >= 2) tc_wait(&kempty[st], ((n >> 1) - 1) & 1, &failed);
#pragma unroll
        for (int i = 0; i < PER_T; ++i) {
          const int p = ct + i * PA_CONV * 32;
          widen(kr[i], ksm + st * OPB, p / (D / 16), p % (D / 16));
        }
        if (ct < 8) {
          sscale[n & 3][ct] = make_float2(ksn, lvn);
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive_local(&kfull[st]);
        if (n >= 2) tc_wait(&vempty[st], ((n >> 1) - 1) & 1, &failed);
#pragma unroll
        for (int i = 0; i < PER_T; ++i) {
          const int p = ct + i * PA_CONV * 32, t = p / (D / 16), cc = p % (D / 16);
          uint32_t u[4] = {vr[i].x, vr[i].y, vr[i].z, vr[i].w};
          uint32_t any = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) any |= (u[e] & 0x7f7f7f7fu) + 0x01010101u;  // a byte of 0x7f carries into its sign
          if (any & 0x80808080u) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t nan = __vcmpeq4(u[e] & 0x7f7f7f7fu, 0x7f7f7f7fu);
              for (int z = 0; z < 4; ++z)
                if ((nan >> (8 * z)) & 1u) atomicMin(&nan_from[cc * 16 + 4 * e + z], j * PA_KT + t);
              u[e] &= ~nan;
            }
          }
          widen(make_uint4(u[0], u[1], u[2], u[3]), vsm + st * OPB, t, cc);
        }
        if (j + 1 < nt) fetch(j + 1);
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive_local(&vfull[st]);
      }
    } else if (lane == 0) {
      // ---- issues the products: scores of tile j follow the weighted values of tile j - 1, query tiles in turn
      constexpr uint32_t is = tc_idesc(false, PA_KT), io = tc_idesc(false, D) | (1u << 16);  // values: columns lie together
      constexpr uint32_t v_hi = (1024u >> 4) | (1u << 14) | (2u << 29);
      tc_wait(&qready, groups & 1, &failed);
      auto weigh = [&](int q, int j) {
        const uint32_t n = tiles + j, st = n & 1;
        tc_wait(&pready[q], scount[q] & 1, &failed);
        ++scount[q];
        if (q == 0) tc_wait(&vfull[st], (n >> 1) & 1, &failed);
        tc_after_sync();
        if (*(volatile int*)&failed) return;
        // panels of 64 columns are 16 KB apart, groups of 8 tokens 1 KB
        const uint32_t v0 = ((saddr(vsm + st * OPB) >> 4) & 0x3fffu) | ((128u * 128u >> 4) << 16);
#pragma unroll
        for (int s = 0; s < PA_KT / 16; ++s) tc_mma_ts(o_at[q], s_at[q] + 8 * s, v0 + s * (2048 / 16), v_hi, io, j > 0 || s > 0);
        if (q == nq - 1) tc_commit(&vempty[st]);
      };
      for (int j = 0; j < nt; ++j) {
        const uint32_t n = tiles + j, st = n & 1;
        tc_wait(&kfull[st], (n >> 1) & 1, &failed);
        for (int q = 0; q < nq; ++q) {
          if (j > 0) weigh(q, j - 1);
          tc_after_sync();
          if (*(volatile int*)&failed) break;
          const uint32_t q0 = tc_desc_lo(saddr(qs + q * OPB)), k0 = tc_desc_lo(saddr(ksm + st * OPB));
#pragma unroll
          for (int s = 0; s < D / 16; ++s) {
            const uint32_t off = (uint32_t)((s >> 2) * (128 * 128) + (s & 3) * 32) / 16;
            tc_mma_ss(s_at[q], q0 + off, TC_DESC_HI, k0 + off, TC_DESC_HI, is, s > 0);
          }
          tc_commit(&sfull[q]);
          if (q == nq - 1) tc_commit(&kempty[st]);
        }
      }
      for (int q = 0; q < nq; ++q) {
        weigh(q, nt - 1);
        tc_commit(&ofull[q]);
      }
      if (nq == 1) tc_commit(&ofull[1]);  // its phase goes with the groups
    }
    __syncwarp();
    tiles += nt;
    ++groups;
    __syncthreads();
  }
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

}  // namespace lss
