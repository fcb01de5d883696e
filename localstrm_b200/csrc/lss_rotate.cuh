// lss_rotate.cuh — norms of queries and keys for each head, with the position rotation in the same pass.
#pragma once

#include <type_traits>

#include "lss_kvcache.cuh"

namespace lss {

constexpr int RO_NT = 256;
constexpr int RO_ST = 4;  // heads on their way to a team

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

// N consecutive values (16 bytes, or one) as loaded, and as f32.
template <int DT, int N>
struct RoVec {
  uint4 v;
  __device__ __forceinline__ void get(float (&f)[N]) const {
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if constexpr (DT == LSS_DTYPE_F32) {
        f[q] = __uint_as_float(u[q]);
      } else if constexpr (DT == LSS_DTYPE_BF16) {
        f[2 * q] = __uint_as_float(u[q] << 16);
        f[2 * q + 1] = __uint_as_float(u[q] & 0xffff0000u);
      } else {
        const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&u[q]));
        f[2 * q] = t.x;
        f[2 * q + 1] = t.y;
      }
    }
  }
  static __device__ __forceinline__ void store(void* p, int64_t i, const float (&f)[N]) {
    uint32_t u[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if constexpr (DT == LSS_DTYPE_F32) {
        u[q] = __float_as_uint(f[q]);
      } else if constexpr (DT == LSS_DTYPE_BF16) {
        const __nv_bfloat162 t = __floats2bfloat162_rn(f[2 * q], f[2 * q + 1]);
        u[q] = *reinterpret_cast<const uint32_t*>(&t);
      } else {
        const __half2 t = __floats2half2_rn(f[2 * q], f[2 * q + 1]);
        u[q] = *reinterpret_cast<const uint32_t*>(&t);
      }
    }
    *reinterpret_cast<uint4*>(reinterpret_cast<char*>(p) + i * (16 / N)) = make_uint4(u[0], u[1], u[2], u[3]);
  }
};
template <int DT>
struct RoVec<DT, 1> {
  float v;
  __device__ __forceinline__ void load(const void* p, int64_t i) {
    v = DT == LSS_DTYPE_F32    ? reinterpret_cast<const float*>(p)[i]
        : DT == LSS_DTYPE_BF16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i])
                               : __half2float(reinterpret_cast<const __half*>(p)[i]);
  }
  __device__ __forceinline__ void get(float (&f)[1]) const { f[0] = v; }
  static __device__ __forceinline__ void store(void* p, int64_t i, const float (&f)[1]) {
    if (DT == LSS_DTYPE_F32) reinterpret_cast<float*>(p)[i] = f[0];
    else if (DT == LSS_DTYPE_BF16) reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(f[0]);
    else reinterpret_cast<__half*>(p)[i] = __float2half_rn(f[0]);
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
// the fraction.  Less its whole part it is exact to 2^-33 or so, and sincospi takes it from there.  A CTA takes TK tokens,
// turns each of their (token, frequency) into cosine and sine once, and has RO_NT / L / TK teams of L lanes per token. A lane
// holds 2 N values that turn with each other, so that no value moves between lanes but for the sum of squares, and for
// all of its team's heads, the queries' and then the keys', keeps the factors of a value and of its partner, w cos
// and +-w sin, in registers.
// Measured: 8,192 tokens of 32 + 8 heads of 128 in bf16, 168 MB: alone with cold caches and launch 39 us, one call behind the
// other 34 to 36 (4.7 to 5.0 TB/s of its own bytes, 0.71 to 0.76 of the copy rate; counters see 3.5 TB/s of DRAM traffic, 0.53,
// as not all results have left the L2 cache when it ends); 4,096 in f32 37 and 30 us, one token of 16 heads of 64 8 and 4 us.
// Not HBM bounds it but the instructions (some 190 per warp and four heads, 19 million in the first case, 54 % of the issue
// slots), their waits for shared memory and fixed latencies, and the start of each CTA (weights, sines: about four heads' time),
// which three CTAs per SM hide from each other.  With half the bytes per head the starts weigh twice: 40 heads of 64 25 and
// 17 us (floor 12.8); rows that are not on 16 bytes go value by value: 1,000 tokens of 40 heads of 66 37 and 24 us (1.6).
// One token per CTA with weights and sines in shared memory: 57 us.
template <int DT, int N, int L, bool PAIRS>  // PAIRS: interleaved
__global__ void __launch_bounds__(RO_NT, N > 1 ? 3 : 2) lss_rotate_kernel(RotateArgs a, int tk) {
  constexpr int NU = N > 1 ? 1 : 8;   // units of 2 N values that a lane holds: dim <= 2 N L NU
  constexpr int ST = N > 1 ? RO_ST : 1;
  constexpr int ES = DT == LSS_DTYPE_F32 ? 4 : 2;
  extern __shared__ __align__(16) float ro_sm[];
  uint4* ring = reinterpret_cast<uint4*>(ro_sm);                  // [ST][2][RO_NT]: each thread's own
  float* wsm = ro_sm + (N > 1 ? ST * 2 * RO_NT * 4 : 0);          // [2][dim]
  float2* turn = reinterpret_cast<float2*>(wsm + 2 * a.dim);      // [tk][half] cosine, sine
  const int tid = threadIdx.x, D = a.dim, half = a.half;
  const int t0 = blockIdx.x * tk, nt = min(tk, a.T - t0);
  const int lane = tid % L, teams = RO_NT / L / tk, t = tid / L / teams, h0 = tid / L - t * teams;
  const int hq = a.side[0].heads, hk = a.side[1].heads;
  // The unit's two groups of N values: where they lie (neighbouring lanes' groups lie together), and whether they turn.
  // Halves: a group turns with the other one of the unit, and units behind the last turned one halve the rest.
  auto at0 = [&](int i) {
    const int u = (lane + i * L) * N;
    return PAIRS ? (N > 1 ? u : 2 * u) : u < half ? u : u + half;
  };
  auto at1 = [&](int i) {
    const int u = (lane + i * L) * N;
    return PAIRS ? (N > 1 ? u + D / 2 : 2 * u + 1) : u < half ? u + half : u + D / 2;
  };
  auto in = [&](int i) { return 2 * (lane + i * L) * N < D; };
  auto turned0 = [&](int i) { return PAIRS ? at0(i) < 2 * half : (lane + i * L) * N < half; };
  auto turned1 = [&](int i) { return PAIRS ? at1(i) < 2 * half : (lane + i * L) * N < half; };
  // The team's heads, every teams-th of the queries' and then of the keys'.
  const char* src = nullptr;  // the lane's first group of the head that is fetched next
  int64_t step = 0;
  int side = -1, left = 0;
  auto turn_to = [&]() {  // the next side with a head of the team
    while (left <= 0 && side < 1) {
      const RotateSide& s = a.side[++side];
      left = t < nt ? (s.heads - h0 + teams - 1) / teams : 0;
      src = reinterpret_cast<const char*>(s.x) + ((int64_t)(t0 + t) * s.x_st + (int64_t)h0 * s.x_sh + at0(0)) * ES;
      step = (int64_t)teams * s.x_sh * ES;
    }
  };
  turn_to();
  RoVec<DT, N> x0[NU], x1[NU];
  constexpr uint32_t STAGE = 2 * RO_NT * 16;
  const uint32_t mine = saddr(ring + tid);
  const int other = (at1(0) - at0(0)) * ES;
  auto load = [&](uint32_t stage) {
    if (left > 0) {
      if constexpr (N > 1) {
        if (in(0)) {
          cp_async16(mine + stage, src);
          cp_async16(mine + stage + RO_NT * 16, src + other);
        }
      } else {
#pragma unroll
        for (int i = 0; i < NU; ++i)
          if (in(i)) {
            x0[i].load(src, at0(i) - at0(0));
            x1[i].load(src, at1(i) - at0(0));
          }
      }
      src += step;
      if (--left == 0) turn_to();
    }
    if (N > 1) cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < (ST > 1 ? ST - 1 : 1); ++i) load(i * STAGE);
  for (int i = tid; i < 2 * D; i += RO_NT) {
    const void* w = a.side[i >= D].w;
    wsm[i] = w ? ro_weight(w, a.w_dtype, i >= D ? i - D : i) : 1.0f;
  }
  for (int i = tid; i < nt * half; i += RO_NT) {
    const int u = i / half, f = i - u * half;
    const double turns = (double)a.positions[t0 + u] * ((double)a.freqs[f] * 0.15915494309189535);
    float s, c;
    sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
    turn[i] = make_float2(c, s);
  }
  __syncthreads();
  if (t >= nt) return;
  const unsigned team = L == 32 ? 0xffffffffu : ((1u << (L & 31)) - 1u) << ((tid & 31) / L * L);
  const float per_dim = 1.0f / (float)D;
  uint32_t stage = 0;
#pragma unroll 1
  for (int which = 0; which < 2; ++which) {
    const bool norm = (which ? a.side[1].w : a.side[0].w) != nullptr;
    const int64_t y_sh = which ? a.side[1].y_sh : a.side[0].y_sh;
    const int end = which ? hk : hq;
    char* dst = reinterpret_cast<char*>(which ? a.side[1].y : a.side[0].y) +
                ((int64_t)(t0 + t) * (which ? a.side[1].y_st : a.side[0].y_st) + h0 * y_sh + at0(0)) * ES;
    const int64_t dst_step = teams * y_sh * ES;
    // Factors of the value itself (p) and of its partner (q): a value of the other group, or its neighbour.
    float p0[NU][N], p1[NU][N], q0[NU][N], q1[NU][N];
#pragma unroll
    for (int i = 0; i < NU; ++i)
      if (in(i)) {
        const float* w = wsm + which * D;
        auto take = [&](float* to, const float* from, int n) {
          if constexpr (N > 1) {
#pragma unroll
            for (int e = 0; e < n; e += 4) *reinterpret_cast<float4*>(to + e) = *reinterpret_cast<const float4*>(from + e);
          } else {
#pragma unroll
            for (int e = 0; e < n; ++e) to[e] = from[e];
          }
        };
        take(p0[i], w + at0(i), N);
        take(p1[i], w + at1(i), N);
        float cs[2 * N];  // cosine, sine of the group's frequencies
        auto pairs = [&](float (&p)[N], float (&q)[N], int at) {
          take(cs, reinterpret_cast<const float*>(turn + t * half + at / 2), N);
#pragma unroll
          for (int e = 0; e < N; e += 2) {
            const int o = e + (N > 1);
            q[e] = -p[o] * cs[e + (N > 1)];
            q[o] = p[e] * cs[e + (N > 1)];
            p[e] *= cs[e];
            p[o] *= cs[e];
          }
        };
        if (PAIRS && N > 1) {
          if (turned0(i)) pairs(p0[i], q0[i], at0(i));
          if (turned1(i)) pairs(p1[i], q1[i], at1(i));
        } else if (turned0(i)) {
          take(cs, reinterpret_cast<const float*>(turn + t * half + (lane + i * L) * N), 2 * N);
#pragma unroll
          for (int e = 0; e < N; ++e) {
            q0[i][e] = -p1[i][e] * cs[2 * e + 1];
            q1[i][e] = p0[i][e] * cs[2 * e + 1];
            p0[i][e] *= cs[2 * e];
            p1[i][e] *= cs[2 * e];
          }
        }
      }
    auto rows = [&](auto all_c) {
      [[maybe_unused]] constexpr bool ALL = decltype(all_c)::value;  // every value turns
#pragma unroll 1
      for (int h = h0; h < end; h += teams, dst += dst_step) {
        float y0[NU][N], y1[NU][N];
        if constexpr (N > 1) {  // the place of the head before is free: what it held is in registers
          load((stage - STAGE) & (ST * STAGE - 1));
          cp_async_wait_group<ST - 1>();
          x0[0].v = *reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(ring + tid) + stage);
          x1[0].v = *reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(ring + tid) + stage + RO_NT * 16);
          stage = (stage + STAGE) & (ST * STAGE - 1);
        }
#pragma unroll
        for (int i = 0; i < NU; ++i) {
          if (in(i)) {
            x0[i].get(y0[i]);
            x1[i].get(y1[i]);
          } else {
#pragma unroll
            for (int e = 0; e < N; ++e) y0[i][e] = y1[i][e] = 0.0f;
          }
        }
        if constexpr (N == 1) load(0);
        float r = 1.0f;
        if (norm) {
          float sum = 0.0f;
          if constexpr (N > 1) {
            float2 s2 = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int e = 0; e < N; e += 2) {
              const float2 v = make_float2(y0[0][e], y0[0][e + 1]), w = make_float2(y1[0][e], y1[0][e + 1]);
              s2 = fma2(w, w, fma2(v, v, s2));
            }
            sum = s2.x + s2.y;
          } else {
#pragma unroll
            for (int i = 0; i < NU; ++i) sum = fmaf(y0[i][0], y0[i][0], fmaf(y1[i][0], y1[i][0], sum));
          }
#pragma unroll
          for (int o = 1; o < L; o <<= 1) sum += __shfl_xor_sync(team, sum, o);
          r = rsqrtf(fmaf(sum, per_dim, a.eps));
        }
#pragma unroll
        for (int i = 0; i < NU; ++i)
          if (in(i)) {
            float z0[N], z1[N];
            if constexpr (N > 1) {
              const bool on0 = ALL || turned0(i), on1 = ALL || turned1(i);
#pragma unroll
              for (int e = 0; e < N; e += 2) {
                const float2 b0 = mul2(make_float2(y0[i][e], y0[i][e + 1]), make_float2(r, r));
                const float2 b1 = mul2(make_float2(y1[i][e], y1[i][e + 1]), make_float2(r, r));
                float2 v0 = mul2(b0, make_float2(p0[i][e], p0[i][e + 1])), v1 = mul2(b1, make_float2(p1[i][e], p1[i][e + 1]));
                if (on0) v0 = fma2(PAIRS ? make_float2(b0.y, b0.x) : b1, make_float2(q0[i][e], q0[i][e + 1]), v0);
                if (on1) v1 = fma2(PAIRS ? make_float2(b1.y, b1.x) : b0, make_float2(q1[i][e], q1[i][e + 1]), v1);
                z0[e] = v0.x;
                z0[e + 1] = v0.y;
                z1[e] = v1.x;
                z1[e + 1] = v1.y;
              }
            } else {
              const float b0 = y0[i][0] * r, b1 = y1[i][0] * r;
              z0[0] = b0 * p0[i][0];
              z1[0] = b1 * p1[i][0];
              if (turned0(i)) {
                z0[0] = fmaf(b1, q0[i][0], z0[0]);
                z1[0] = fmaf(b0, q1[i][0], z1[0]);
              }
            }
            RoVec<DT, N>::store(dst, at0(i) - at0(0), z0);
            RoVec<DT, N>::store(dst, at1(i) - at0(0), z1);
          }
      }
    };
    if (N > 1 && 2 * half == D) rows(std::true_type{}); else rows(std::false_type{});
  }
}

}  // namespace lss
