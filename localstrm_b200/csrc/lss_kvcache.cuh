// lss_kvcache.cuh — write of a step's keys and values into a paged cache of 8-bit values (e4m3)
// with one scale per block and key head.
#pragma once

#include "lss_common.cuh"

namespace lss {

constexpr int KV_NT = 256;
constexpr int KV_HOLD = 8;      // groups of eight values that a lane keeps between its two passes
constexpr float E4M3_MAX = 448.0f;

struct AppendArgs {
  const void* k;
  const void* v;
  int64_t k_st, k_sh, v_st, v_sh;  // strides in elements: token, head
  uint8_t* kc;                     // [num_blocks][heads][block_size][dim]
  uint8_t* vc;
  float* ks;                       // [num_blocks][heads]
  float* vs;
  int num_blocks, heads, bs_shift, dim;
  const int32_t* table;
  int64_t table_stride;
  int width;
  const int32_t* starts;
  const int32_t* granted;
  const int32_t* lens;
  int B, T;
  int aligned;                     // every group of eight values starts on a 16-byte boundary
};

// Eight consecutive values as loaded: 16 bytes of 16-bit values or 32 of f32.
template <int DT>
struct Vec8 {
  uint4 w[DT == LSS_DTYPE_F32 ? 2 : 1];
  __device__ __forceinline__ void load(const void* p, int64_t i, bool aligned) {
    if (DT == LSS_DTYPE_F32) {
      const float* f = reinterpret_cast<const float*>(p) + i;
      if (aligned) {
        w[0] = __ldg(reinterpret_cast<const uint4*>(f));
        w[DT == LSS_DTYPE_F32 ? 1 : 0] = __ldg(reinterpret_cast<const uint4*>(f) + 1);
      } else {
        uint32_t* u = reinterpret_cast<uint32_t*>(w);
#pragma unroll
        for (int q = 0; q < (DT == LSS_DTYPE_F32 ? 8 : 0); ++q) u[q] = __float_as_uint(f[q]);
      }
    } else {
      const uint16_t* h = reinterpret_cast<const uint16_t*>(p) + i;
      if (aligned) {
        w[0] = __ldg(reinterpret_cast<const uint4*>(h));
      } else {
        uint32_t* u = reinterpret_cast<uint32_t*>(w);
#pragma unroll
        for (int q = 0; q < 4; ++q) u[q] = (uint32_t)h[2 * q] | ((uint32_t)h[2 * q + 1] << 16);
      }
    }
  }
  // Magnitudes as whole numbers (their order is that of the values; not finite ones on top): the
  // larger of `m` and the values', 16-bit types two at a time.
  __device__ __forceinline__ uint32_t top(uint32_t m) const {
    const uint32_t* u = reinterpret_cast<const uint32_t*>(w);
#pragma unroll
    for (int q = 0; q < (DT == LSS_DTYPE_F32 ? 8 : 4); ++q)
      m = DT == LSS_DTYPE_F32 ? max(m, u[q] & 0x7fffffffu) : __vmaxu2(m, u[q] & 0x7fff7fffu);
    return m;
  }
  __device__ __forceinline__ float2 pair(int q) const {  // values 2 q and 2 q + 1
    const uint32_t* u = reinterpret_cast<const uint32_t*>(w);
    if (DT == LSS_DTYPE_F32) return make_float2(get(2 * q), get(2 * q + 1));
    if (DT == LSS_DTYPE_BF16) return make_float2(__uint_as_float(u[q] << 16), __uint_as_float(u[q] & 0xffff0000u));
    return __half22float2(*reinterpret_cast<const __half2*>(u + q));
  }
  __device__ __forceinline__ float get(int q) const {  // q a constant after unrolling
    const uint32_t* u = reinterpret_cast<const uint32_t*>(w);
    if (DT == LSS_DTYPE_F32) return __uint_as_float(u[DT == LSS_DTYPE_F32 ? q : 0]);
    const uint16_t b = (uint16_t)(u[q >> 1] >> ((q & 1) * 16));
    if (DT == LSS_DTYPE_BF16) return __uint_as_float((uint32_t)b << 16);
    return __half2float(__ushort_as_half(b));
  }
};

// Two f32 values to e4m3, to nearest even; beyond +-448 (infinities among them) saturates, NaN stays.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ __half2 e4m3x2_to_half2(uint16_t v) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(v));
  return *reinterpret_cast<__half2*>(&r);
}

// Smallest power of two s with amax <= 448 s, at least 2^-126 (448 = 1.75 * 2^8).
__device__ __forceinline__ float e4m3_scale(float amax) {
  const uint32_t u = __float_as_uint(amax);
  int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u);
  e = max(e, -126);
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

// Rows of [0, n) found by their inclusive sums: the first whose sum exceeds u.
__device__ __forceinline__ int row_of(const int32_t* upto, int n, int u) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (upto[mid] > u) hi = mid; else lo = mid + 1;
  }
  return lo;
}

// A block that this call writes is one unit: the tokens of its row that fall into it, for one head,
// of K or V, by one team of TEAM warps, so that the scale of (block, head) has one writer and no atomics.
// Pass one takes the largest finite magnitude of the new values; the scale becomes
//   s = max(s_old, 2^e),  e the smallest with amax <= 448 * 2^e,
// where s_old counts only if the block keeps tokens of earlier steps; kept values are re-rounded
// (code * s_old / s) where the scale grew.  Powers of two make every division exact, so a value is
// rounded once when it is written and once more for each growth of its block's scale, by at most half
// a step of e4m3 each (2^-4 relative; below 2^-6 s the step is 2^-9 s).
// Up to 2048 TEAM values stay in registers between the passes; what goes beyond is read again, from the
// L2 cache.
// Measured: 24 rows of up to 2,048 new tokens, 8 heads of 128, f16: 39 us (153 MB, 3.9 TB/s, 0.60 of the copy
// rate; a fixed part of some 400 instructions per unit and warp and the rounding bound it), one warp per
// block of 32 tokens 68 us; in f32 (254 MB, half the values held in registers) 60 us; 256 single tokens 6.4 us in a graph.
// Bound by issue and HBM for prompts and by its chain of dependent loads (lengths, table, scale, values) for
// single tokens.
template <int DT, int TEAM>
__global__ void __launch_bounds__(KV_NT, 3) lss_append_kernel(AppendArgs a) {
  constexpr int HOLD = DT == LSS_DTYPE_F32 ? KV_HOLD / 2 : KV_HOLD;
  constexpr uint32_t INF = DT == LSS_DTYPE_F32 ? 0x7f800000u : DT == LSS_DTYPE_BF16 ? 0x7f80u : 0x7c00u;
  extern __shared__ int32_t kv_sm[];
  int32_t* upto = kv_sm;  // [B] inclusive sums of the blocks that the rows write
  __shared__ int scr[KV_NT / 32];
  constexpr int TEAMS = KV_NT / 32 / TEAM, TL = TEAM * 32;
  __shared__ uint32_t found[2][KV_NT / 32];  // the warps' largest magnitudes, two in turn
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int team = tid / TL, tl = tid % TL;
  const int sh = a.bs_shift, bs = 1 << sh, D = a.dim;
  const int64_t room = (int64_t)a.width << sh;
  int units = 0;
  for (int r0 = 0; r0 < a.B; r0 += KV_NT) {
    const int r = r0 + tid;
    int n = 0;
    if (r < a.B) {
      const int g = a.granted[r], len = a.lens[r], s = a.starts[r];
      if (g > 0 && g <= len && len <= room && s >= 0 && (int64_t)s + g <= a.T) n = ((len - 1) >> sh) - ((len - g) >> sh) + 1;
    }
    int x = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) scr[warp] = x;
    __syncthreads();
    int before = 0, tot = 0;
#pragma unroll
    for (int i = 0; i < KV_NT / 32; ++i) {
      if (i < warp) before += scr[i];
      tot += scr[i];
    }
    if (r < a.B) upto[r] = units + before + x;
    units += tot;
  }
  __syncthreads();

  // Items (unit, head, K or V), dealt to the teams of the grid in turn.
  const int per = 2 * a.heads, step = (int)gridDim.x * TEAMS;
  const int it0 = (int)blockIdx.x * TEAMS + team, step_u = step / per, step_w = step - step_u * per;
  // Largest value of the team's threads, the same for all of them (positive f32 values order as their bits do).
  int turn = 0;
  auto team_max = [&](uint32_t v) {
    v = __reduce_max_sync(0xffffffffu, v);
    if (TEAM > 1) {
      if (lane == 0) found[turn][warp] = v;
      asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "n"(TL) : "memory");
#pragma unroll
      for (int i = 0; i < TEAM; ++i) v = max(v, found[turn][team * TEAM + i]);
      turn ^= 1;
    }
    return v;
  };
  int u = it0 / per, which = it0 - u * per;
  // The thread's places in a unit: group of eight e = tl + TL i is (token, column) = (e / d8, e % d8).
  const int d8 = D >> 3, tok0 = tl / d8, col0 = tl - tok0 * d8, step_t = TL / d8, step_c = TL - step_t * d8;
  while (u < units) {
    const int head = which >> 1;
    const bool is_v = which & 1;
    const int r = row_of(upto, a.B, u);
    const int len = a.lens[r], old = len - a.granted[r];
    const int j = (old >> sh) + u - (r > 0 ? upto[r - 1] : 0);
    const int lo = max(old - (j << sh), 0), hi = min(len - (j << sh), bs);  // new tokens: offsets [lo, hi)
    const int page = a.table[r * a.table_stride + j];
    const int tok = a.starts[r] + (j << sh) + lo - old;
    u += step_u;
    which += step_w;
    if (which >= per) {
      which -= per;
      ++u;
    }
    if ((unsigned)page >= (unsigned)a.num_blocks) continue;
    const void* x = is_v ? a.v : a.k;
    const int64_t st = is_v ? a.v_st : a.k_st, src = (int64_t)tok * st + head * (is_v ? a.v_sh : a.k_sh);
    const int64_t ph = (int64_t)page * a.heads + head;
    uint8_t* dst = (is_v ? a.vc : a.kc) + (ph << sh) * D;
    float* sp = (is_v ? a.vs : a.ks) + ph;
    const int n = (hi - lo) * d8;
    Vec8<DT> keep[HOLD];
    int t = tok0, c = col0;
    auto next = [&]() {
      t += step_t;
      c += step_c;
      if (c >= d8) {
        c -= d8;
        ++t;
      }
    };
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < HOLD; ++i) {
      if (TL * i < n) {
        if (tl + TL * i < n) keep[i].load(x, src + t * st + c * 8, a.aligned);
        next();
      }
    }
    const float was = lo > 0 ? *sp : 0.0f;
    const int t1 = t, c1 = c;
#pragma unroll
    for (int i = 0; i < HOLD; ++i)
      if (TL * i < n && tl + TL * i < n) top = keep[i].top(top);
#pragma unroll 4
    for (int e = tl + TL * HOLD; e < n; e += TL) {
      Vec8<DT> w;
      w.load(x, src + t * st + c * 8, a.aligned);
      top = w.top(top);
      next();
    }
    if (DT != LSS_DTYPE_F32) top = max(top & 0xffffu, top >> 16);
    top = team_max(top);
    float amax;
    if (top < INF) {
      amax = DT == LSS_DTYPE_F32 ? __uint_as_float(top) : DT == LSS_DTYPE_BF16 ? __uint_as_float(top << 16) : __half2float(__ushort_as_half((uint16_t)top));
    } else {  // some value is not finite: the others decide, read again one by one
      amax = 0.0f;
      t = tok0, c = col0;
      for (int e = tl; e < n; e += TL) {
        Vec8<DT> w;
        w.load(x, src + t * st + c * 8, a.aligned);
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          const float f = fabsf(w.get(q));
          if (f <= FLT_MAX) amax = fmaxf(amax, f);
        }
        next();
      }
      amax = __uint_as_float(team_max(__float_as_uint(amax)));
    }
    const float s = fmaxf(was, e4m3_scale(amax));
    const bool pow2 = (__float_as_uint(s) & 0x7fffffu) == 0u;
    const float inv = __frcp_rn(s);
    auto store = [&](const Vec8<DT>& w, int e) {
      float f[8];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float2 v = w.pair(q);
        f[2 * q] = v.x * inv;
        f[2 * q + 1] = v.y * inv;
      }
      if (!pow2) {  // a scale of the caller's own
#pragma unroll
        for (int q = 0; q < 8; ++q) f[q] = __fdiv_rn(w.get(q), s);
      }
      uint2 o;
      o.x = e4m3x2(f[0], f[1]) | (e4m3x2(f[2], f[3]) << 16);
      o.y = e4m3x2(f[4], f[5]) | (e4m3x2(f[6], f[7]) << 16);
      *reinterpret_cast<uint2*>(dst + (lo * D + e * 8)) = o;
    };
#pragma unroll
    for (int i = 0; i < HOLD; ++i)
      if (TL * i < n && tl + TL * i < n) store(keep[i], tl + TL * i);
    t = t1, c = c1;
#pragma unroll 4
    for (int e = tl + TL * HOLD; e < n; e += TL) {
      Vec8<DT> w;
      w.load(x, src + t * st + c * 8, a.aligned);
      store(w, e);
      next();
    }
    if (lo > 0 && s != was) {  // kept tokens, rounded again to the larger step
      const float ratio = __fdiv_rn(was, s);
#pragma unroll 4
      for (int e = tl; e < lo * d8; e += TL) {
        uint2* at = reinterpret_cast<uint2*>(dst + e * 8);
        const uint2 k8 = *at;
        const uint32_t in[4] = {k8.x & 0xffffu, k8.x >> 16, k8.y & 0xffffu, k8.y >> 16};
        uint32_t out[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float2 f = __half22float2(e4m3x2_to_half2((uint16_t)in[q]));
          out[q] = e4m3x2(f.x * ratio, f.y * ratio);
        }
        *at = make_uint2(out[0] | (out[1] << 16), out[2] | (out[3] << 16));
      }
    }
    if (tl == 0 && !(s == was)) *sp = s;
  }
}

}  // namespace lss
