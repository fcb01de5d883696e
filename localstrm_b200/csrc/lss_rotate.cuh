// lss_rotate.cuh — norms of queries and keys for each head, with the position rotation in the same pass.
#pragma once

#include "lss_kvcache.cuh"

namespace lss {

constexpr int RO_NT = 256;

struct RotateSide {
  const void* x;
  void* y;
  const void* w;                 // [dim] or NULL: no norm
  int64_t x_st, x_sh, y_st, y_sh;  // strides in elements: token, head
  int heads;
};
struct RotateArgs {
  RotateSide side[2];            // queries, keys
  const int32_t* positions;      // [T]
  const float* freqs;            // [half]
  int T, dim, half, w_dtype, interleaved;
  float eps;
};

// N consecutive values (N 1 or 8) as f32.
template <int DT, int N>
struct RoVec {
  float f[N];
  __device__ __forceinline__ void load(const void* p, int64_t i) {
    if constexpr (N == 8) {
      Vec8<DT> v;
      v.load(p, i, true);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float2 t = v.pair(q);
        f[2 * q] = t.x;
        f[2 * q + 1] = t.y;
      }
    } else {
      f[0] = DT == LSS_DTYPE_F32    ? reinterpret_cast<const float*>(p)[i]
             : DT == LSS_DTYPE_BF16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i])
                                    : __half2float(reinterpret_cast<const __half*>(p)[i]);
    }
  }
  __device__ __forceinline__ void store(void* p, int64_t i) const {
    if constexpr (N == 8) {
      if constexpr (DT == LSS_DTYPE_F32) {
        float4* o = reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + i);
        o[0] = make_float4(f[0], f[1], f[2], f[3]);
        o[1] = make_float4(f[4], f[5], f[6], f[7]);
      } else {
        uint32_t u[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if constexpr (DT == LSS_DTYPE_BF16) {
            const __nv_bfloat162 v = __floats2bfloat162_rn(f[2 * q], f[2 * q + 1]);
            u[q] = *reinterpret_cast<const uint32_t*>(&v);
          } else {
            const __half2 v = __floats2half2_rn(f[2 * q], f[2 * q + 1]);
            u[q] = *reinterpret_cast<const uint32_t*>(&v);
          }
        }
        *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p) + i) = make_uint4(u[0], u[1], u[2], u[3]);
      }
    } else {
      if (DT == LSS_DTYPE_F32) reinterpret_cast<float*>(p)[i] = f[0];
      else if (DT == LSS_DTYPE_BF16) reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(f[0]);
      else reinterpret_cast<__half*>(p)[i] = __float2half_rn(f[0]);
    }
  }
};

__device__ __forceinline__ float ro_weight(const void* w, int dtype, int i) {
  return dtype == LSS_DTYPE_F32    ? reinterpret_cast<const float*>(w)[i]
         : dtype == LSS_DTYPE_BF16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(w)[i])
                                   : __half2float(reinterpret_cast<const __half*>(w)[i]);
}

// y = x / sqrt(mean(x^2) + eps) * w for each head (where there is a weight), then each pair (a, b) of the first
// 2 half values turned by the angle positions[t] * freqs[i]:  (a cos - b sin, b cos + a sin); pairs are (i, i + half),
// or (2 i, 2 i + 1) where interleaved.  Squares, sums and products are f32, one rounding at the end.
//
// The angle in turns, position * freq / 2 pi, is a double: of a position of 10^6 f32 would leave two digits of
// the fraction.  Less its whole part it is exact to 2^-33 or so, and sincospi takes it from there.  A CTA takes TK tokens and
// has every (token, frequency) turned into cosine and sine once, for all heads: 8 sines of a lane would cost
// more than its two 16-byte loads.  Then L lanes take a head, each 2 N values that turn with each other, so that no
// value moves between lanes but for the sum of squares.
template <int DT, int N, int L>
__global__ void __launch_bounds__(RO_NT) lss_rotate_kernel(RotateArgs a, int tk) {
  constexpr int NU = N == 8 ? 1 : 8;  // units of 2 N values that a lane holds: dim <= 2 N L NU
  extern __shared__ float ro_sm[];
  float2* turn = reinterpret_cast<float2*>(ro_sm);        // [tk][half] cosine, sine
  float* wq = ro_sm + 2 * tk * a.half;                    // [2][dim]
  const int tid = threadIdx.x, D = a.dim, half = a.half;
  const int t0 = blockIdx.x * tk, nt = min(tk, a.T - t0);
  const int hq = a.side[0].heads, hs = hq + a.side[1].heads, items = nt * hs;
  const int lane = tid % L;
  // The unit's two groups of N values, and the frequency of the first.
  int at0[NU], at1[NU], fr[NU];  // fr < 0: not turned; at0 < 0: nothing
#pragma unroll
  for (int i = 0; i < NU; ++i) {
    const int u = lane + i * L;
    const bool turned = u * N < half;
    at0[i] = u * 2 * N >= D ? -1 : turned && !a.interleaved ? u * N : u * 2 * N;
    at1[i] = turned && !a.interleaved ? u * N + half : u * 2 * N + N;
    fr[i] = turned ? u * N : -1;
  }
  RoVec<DT, N> x0[NU], x1[NU];
  auto load = [&](int it) {
    const int t = it / hs, h = it - t * hs, which = h >= hq;
    const RotateSide& s = a.side[which];
    const int64_t at = (int64_t)(t0 + t) * s.x_st + (int64_t)(h - (which ? hq : 0)) * s.x_sh;
#pragma unroll
    for (int i = 0; i < NU; ++i)
      if (at0[i] >= 0) {
        x0[i].load(s.x, at + at0[i]);
        x1[i].load(s.x, at + at1[i]);
      }
  };
  int it = tid / L;
  if (it < items) load(it);
  for (int i = tid; i < nt * half; i += RO_NT) {
    const int t = i / half, f = i - t * half;
    const double turns = (double)a.positions[t0 + t] * ((double)a.freqs[f] * 0.15915494309189535);
    float s, c;
    sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
    turn[i] = make_float2(c, s);
  }
  for (int i = tid; i < 2 * D; i += RO_NT) {
    const void* w = a.side[i >= D].w;
    if (w) wq[i] = ro_weight(w, a.w_dtype, i >= D ? i - D : i);
  }
  __syncthreads();
  const unsigned team = L == 32 ? 0xffffffffu : ((1u << (L & 31)) - 1u) << ((tid & 31) / L * L);
  while (it < items) {
    const int t = it / hs, h = it - t * hs, which = h >= hq;
    const RotateSide& s = a.side[which];
    float y0[NU][N], y1[NU][N];
#pragma unroll
    for (int i = 0; i < NU; ++i)
#pragma unroll
      for (int e = 0; e < N; ++e) {
        y0[i][e] = at0[i] >= 0 ? x0[i].f[e] : 0.0f;
        y1[i][e] = at0[i] >= 0 ? x1[i].f[e] : 0.0f;
      }
    it += RO_NT / L;
    if (it < items) load(it);
    if (s.w) {
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < NU; ++i)
#pragma unroll
        for (int e = 0; e < N; ++e) sum = fmaf(y0[i][e], y0[i][e], fmaf(y1[i][e], y1[i][e], sum));
#pragma unroll
      for (int o = 1; o < L; o <<= 1) sum += __shfl_xor_sync(team, sum, o);
      const float r = rsqrtf(sum / (float)D + a.eps);
      const float* w = wq + which * D;
#pragma unroll
      for (int i = 0; i < NU; ++i)
        if (at0[i] >= 0) {
#pragma unroll
          for (int e = 0; e < N; ++e) {
            y0[i][e] *= r * w[at0[i] + e];
            y1[i][e] *= r * w[at1[i] + e];
          }
        }
    }
    const int64_t at = (int64_t)(t0 + t) * s.y_st + (int64_t)(h - (which ? hq : 0)) * s.y_sh;
#pragma unroll
    for (int i = 0; i < NU; ++i)
      if (at0[i] >= 0) {
        RoVec<DT, N> o0, o1;
#pragma unroll
        for (int e = 0; e < N; ++e) {
          o0.f[e] = y0[i][e];
          o1.f[e] = y1[i][e];
        }
        if (fr[i] >= 0) {
          const float2* cs = turn + t * half + fr[i];
          if (N > 1 && a.interleaved) {
            // values 2 j, 2 j + 1 of the sixteen are a pair
#pragma unroll
            for (int e = 0; e < N; e += 2) {
              const float2 p = cs[e / 2], q = cs[N / 2 + e / 2];
              o0.f[e] = y0[i][e] * p.x - y0[i][e + (N > 1)] * p.y;
              o0.f[e + (N > 1)] = y0[i][e + (N > 1)] * p.x + y0[i][e] * p.y;
              o1.f[e] = y1[i][e] * q.x - y1[i][e + (N > 1)] * q.y;
              o1.f[e + (N > 1)] = y1[i][e + (N > 1)] * q.x + y1[i][e] * q.y;
            }
          } else {
#pragma unroll
            for (int e = 0; e < N; ++e) {
              o0.f[e] = y0[i][e] * cs[e].x - y1[i][e] * cs[e].y;
              o1.f[e] = y1[i][e] * cs[e].x + y0[i][e] * cs[e].y;
            }
          }
        }
        o0.store(s.y, at + at0[i]);
        o1.store(s.y, at + at1[i]);
      }
  }
}

}  // namespace lss
