// lss_int4.cuh — products of a few rows with a matrix of 4-bit weights and group scales.
#pragma once

#include "lss_common.cuh"

namespace lss {

constexpr int I4_NW = 16;          // warps per CTA
constexpr int I4_NT = I4_NW * 32;
constexpr int I4_ST = 4;           // stages of the copy ring per warp
constexpr int I4_ROWS = 8;         // rows of x that one pass takes
constexpr int I4_KB = 128;         // columns per unit

struct Int4Args {
  const void* x;
  int64_t x_stride;
  int rows, K, N;
  const uint8_t* packed;   // [N][K / 2], the even column in the low four bits
  const uint16_t* scales;  // [N][K / group]
  int group, scale_bf16;
  void* y;
  int y_dtype;
  int64_t y_stride;
  int x_aligned;
};

template <bool BF>
__device__ __forceinline__ void mma_16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (BF)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Eight codes of a 32-bit word (columns k .. k+7) as code - 8 in pairs (k, k+4), (k+1, k+5),
// (k+2, k+6), (k+3, k+7).  The four bits go into the mantissa of a number whose unit is 1 (1024 in
// f16, 128 in bf16), so one subtraction gives the exact value.
template <bool BF>
__device__ __forceinline__ void int4_unpack(uint32_t w, uint32_t (&r)[4]) {
  if (BF) {
    const __nv_bfloat162 off = __halves2bfloat162(__ushort_as_bfloat16(0x4308), __ushort_as_bfloat16(0x4308));  // 136
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t u = ((w >> (4 * i)) & 0x000f000fu) | 0x43004300u;
      const __nv_bfloat162 v = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&u), off);
      r[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
  } else {
    const __half2 off = __halves2half2(__ushort_as_half(0x6408), __ushort_as_half(0x6408));    // 1032
    const __half2 six = __halves2half2(__ushort_as_half(0x2c00), __ushort_as_half(0x2c00));    // 1 / 16
    const __half2 off16 = __halves2half2(__ushort_as_half(0xd480), __ushort_as_half(0xd480));  // -72
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t s = w >> (8 * i);
      uint32_t u = (s & 0x000f000fu) | 0x64006400u, v = (s & 0x00f000f0u) | 0x64006400u;
      const __half2 a = __hsub2(*reinterpret_cast<__half2*>(&u), off);
      const __half2 b = __hfma2(*reinterpret_cast<__half2*>(&v), six, off16);
      r[2 * i] = *reinterpret_cast<const uint32_t*>(&a);
      r[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&b);
    }
  }
}

// Copies 4 bytes of which `valid` are read, the rest zero.
__device__ __forceinline__ void cp_async4z(uint32_t dst, const void* src, int valid) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(valid) : "memory");
}
__device__ __forceinline__ void cp_async16z(uint32_t dst, const void* src, int valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid) : "memory");
}

// Where the 16 bytes `q` (32 columns) of row `r` of a unit lie: pieces permuted so that the 8 rows
// that a warp reads at once fall into 8 different bank groups.
__device__ __forceinline__ uint32_t i4_offset(int r, int q) {
  return (uint32_t)((r >> 1) * 128 + (r & 1) * 64 + ((q ^ ((r >> 1) & 3)) << 4));
}

template <int DT>
__device__ __forceinline__ float i4_widen(const void* p, int64_t i) {
  if (DT == LSS_DTYPE_F32) return reinterpret_cast<const float*>(p)[i];
  if (DT == LSS_DTYPE_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(reinterpret_cast<const __half*>(p)[i]);
}

__device__ __forceinline__ void i4_store(const Int4Args& a, int row, int n, float v) {
  const int64_t at = (int64_t)row * a.y_stride + n;
  if (a.y_dtype == LSS_DTYPE_F32) reinterpret_cast<float*>(a.y)[at] = v;
  else if (a.y_dtype == LSS_DTYPE_BF16) reinterpret_cast<__nv_bfloat16*>(a.y)[at] = __float2bfloat16_rn(v);
  else reinterpret_cast<__half*>(a.y)[at] = __float2half_rn(v);
}

// Stages columns [k0, k0 + kn) of `rows` rows of x in shared memory as matrix operands: for each 32
// columns, row and quarter of them the 8 values in the order of int4_unpack's pairs (16 bytes).
// f32 values become three planes of bf16 that add up to them exactly (8 + 8 + 8 bits, truncated).
template <int DT>
__device__ __forceinline__ void i4_stage_x(const Int4Args& a, int row0, int rows, int k0, int kn, unsigned char* xs) {
  constexpr int P = DT == LSS_DTYPE_F32 ? 3 : 1;
  const int groups = kn >> 3;  // kn is a multiple of 128; columns from K on are zero
  for (int i = threadIdx.x; i < rows * groups; i += blockDim.x) {
    const int r = i / groups, q = i - r * groups, k = k0 + q * 8;
    const int64_t at = (int64_t)(row0 + r) * a.x_stride + k;
    unsigned char* dst = xs + ((int64_t)(q >> 2) * rows + r) * 64 + (q & 3) * 16;
    constexpr int ord[8] = {0, 4, 1, 5, 2, 6, 3, 7};
    if (DT == LSS_DTYPE_F32) {
      float f[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = k < a.K ? reinterpret_cast<const float*>(a.x)[at + e] : 0.0f;
      const int64_t plane = (int64_t)(kn >> 5) * rows * 64;
#pragma unroll
      for (int p = 0; p < P; ++p) {
        uint16_t h[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          h[e] = (uint16_t)(__float_as_uint(f[e]) >> 16);
          // An infinity leaves no rest; a NaN whose payload lies in the low half stays one.
          if (f[e] != f[e]) h[e] |= 0x40;
          const float rest = f[e] - __uint_as_float((uint32_t)h[e] << 16);
          f[e] = fabsf(f[e]) <= FLT_MAX ? rest : 0.0f;
        }
        uint32_t o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = (uint32_t)h[ord[2 * e]] | ((uint32_t)h[ord[2 * e + 1]] << 16);
        *reinterpret_cast<uint4*>(dst + p * plane) = make_uint4(o[0], o[1], o[2], o[3]);
      }
    } else {
      uint16_t h[8];
      const uint16_t* src = reinterpret_cast<const uint16_t*>(a.x) + at;
      if (k < a.K) {  // K is a multiple of 32
        if (a.x_aligned) {
          const uint4 v = __ldg(reinterpret_cast<const uint4*>(src));
          const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int e = 0; e < 8; ++e) h[e] = (uint16_t)(u[e >> 1] >> ((e & 1) * 16));
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) h[e] = src[e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] = 0;
      }
      uint32_t o[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = (uint32_t)h[ord[2 * e]] | ((uint32_t)h[ord[2 * e + 1]] << 16);
      *reinterpret_cast<uint4*>(dst) = make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
}

// y[r, n] = sum_g scale[n, g] * sum_{k in g} x[r, k] (code[n, k] - 8)  for up to 8 rows of x.
//
// A unit is 16 matrix rows times 128 columns (1 KB of codes).  A cluster of ks CTAs takes a range of
// 16-row blocks, each of its CTAs a slice of the columns; inside a CTA the units, row block by row
// block, are cut into equal ranges, one per warp, so that the bytes are spread evenly whatever N and K
// are.  Every warp streams its units through its own ring of asynchronous copies; x lies in shared
// memory as matrix operands for the whole kernel.  The codes are widened to exact 16-bit values of
// x's type (bf16 for f32 x, as three exact parts) and multiplied as the 16-row operand of
// mma.m16n8k16 with f32 sums; the group's sum is then scaled in f32.  Pieces of a row block that was
// cut between warps are added up in shared memory, those between CTAs through distributed shared
// memory, always in the same order.
// Bound by HBM: 0.5 bytes per weight plus the scales.
template <int DT, int SPG>  // SPG: 32-column steps per group (1, 2, or 4 for groups of 128 and more)
__global__ void __launch_bounds__(I4_NT, 1) lss_int4_kernel(Int4Args a, int row0, int rows, int ks) {
  constexpr bool BF = DT != LSS_DTYPE_F16;
  constexpr int P = DT == LSS_DTYPE_F32 ? 3 : 1;
  constexpr int SPU = 4 / SPG;                 // scales per row and unit
  constexpr int STAGE = 1024 + 64 * SPU;
  extern __shared__ __align__(128) unsigned char i4_sm[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
  cg::cluster_group cl = cg::this_cluster();
  const int rank = ks > 1 ? (int)cl.block_rank() : 0;
  const int cluster = blockIdx.x / ks, nclusters = gridDim.x / ks;
  const int NB = (a.N + 15) >> 4, KB = (a.K + I4_KB - 1) / I4_KB, ng = a.K / a.group;
  const int rb0 = (int)((int64_t)NB * cluster / nclusters), rb1 = (int)((int64_t)NB * (cluster + 1) / nclusters);
  const int kb0 = KB * rank / ks, kb1 = KB * (rank + 1) / ks, nk = kb1 - kb0;
  const int nrb = rb1 - rb0, units = nrb * nk;

  // Shared memory: rings, then the pieces (two per warp, 16 x 8 sums each), then the row blocks'
  // sums (clusters only), then x.
  const uint32_t ring = saddr(i4_sm) + (uint32_t)warp * (I4_ST * STAGE);
  float* piece = reinterpret_cast<float*>(i4_sm + I4_NW * I4_ST * STAGE);
  float* sums = piece + I4_NW * 2 * 128;
  unsigned char* xs = reinterpret_cast<unsigned char*>(sums + (ks > 1 ? ((NB + nclusters - 1) / nclusters) * 128 : 0));

  const int u0 = (int)((int64_t)units * warp / I4_NW), u1 = (int)((int64_t)units * (warp + 1) / I4_NW);
  int irb = nk > 0 ? u0 / nk : 0, ikb = nk > 0 ? u0 - irb * nk : 0;  // next unit to fetch
  int iu = u0;
  auto issue = [&](int s) {
    if (iu < u1) {
      const uint32_t dst = ring + (uint32_t)s * STAGE;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int q = lane + 32 * i, r = q >> 2, ch = q & 3;
        const int n = min((rb0 + irb) * 16 + r, a.N - 1);
        const int k = (kb0 + ikb) * I4_KB + ch * 32;
        const bool in = k < a.K;
        cp_async16z(dst + i4_offset(r, ch), a.packed + (int64_t)n * (a.K >> 1) + (in ? k >> 1 : 0), in ? 16 : 0);
      }
      for (int i = lane; i < 16 * SPU; i += 32) {  // the 32-bit word that holds the scale
        const int r = i & 15, q = i >> 4;
        const int n = min((rb0 + irb) * 16 + r, a.N - 1);
        const int k = min((kb0 + ikb) * I4_KB + q * SPG * 32, a.K - 1);
        const int64_t at = (int64_t)n * ng + k / a.group;
        cp_async4z(dst + 1024 + 4 * i, a.scales + (at & ~(int64_t)1), at & 1 ? 4 : 2);
      }
      ++iu;
      if (++ikb == nk) {
        ikb = 0;
        ++irb;
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int s = 0; s < I4_ST - 1; ++s) issue(s);
  i4_stage_x<DT>(a, row0, rows, kb0 * I4_KB, nk * I4_KB, xs);
  __syncthreads();

  float acc[4] = {};
  int rb = nk > 0 ? u0 / nk : 0, kb = nk > 0 ? u0 - rb * nk : 0;
  bool from_start = kb == 0;
  int stage = 0, fill = I4_ST - 1;
  auto emit_full = [&]() {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int n = g + 8 * (e >> 1), r = 2 * c + (e & 1);
      if (ks > 1) {
        sums[rb * 128 + n * 8 + r] = acc[e];
      } else if (r < rows && (rb0 + rb) * 16 + n < a.N) {
        i4_store(a, row0 + r, (rb0 + rb) * 16 + n, acc[e]);
      }
    }
  };
  auto emit_piece = [&](int slot) {
    float* p = piece + (warp * 2 + slot) * 128;
#pragma unroll
    for (int e = 0; e < 4; ++e) p[(g + 8 * (e >> 1)) * 8 + 2 * c + (e & 1)] = acc[e];
  };
  for (int u = u0; u < u1; ++u) {
    cp_async_wait_group<I4_ST - 2>();
    __syncwarp();
    issue(fill);
    fill = fill + 1 == I4_ST ? 0 : fill + 1;
    const uint32_t wt = ring + (uint32_t)stage * STAGE;
    stage = stage + 1 == I4_ST ? 0 : stage + 1;
    float part[4] = {};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t w0, w1, lo[4], hi[4];
      asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w0) : "r"(wt + i4_offset(g, j) + 4 * c) : "memory");
      asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w1) : "r"(wt + i4_offset(g + 8, j) + 4 * c) : "memory");
      int4_unpack<BF>(w0, lo);
      int4_unpack<BF>(w1, hi);
      const uint32_t f0[4] = {lo[0], hi[0], lo[1], hi[1]}, f1[4] = {lo[2], hi[2], lo[3], hi[3]};
#pragma unroll
      for (int p = 0; p < P; ++p) {
        uint4 b = make_uint4(0, 0, 0, 0);
        if (g < rows)
          b = *reinterpret_cast<const uint4*>(xs + (((int64_t)p * nk * 4 + kb * 4 + j) * rows + g) * 64 + c * 16);
        mma_16<BF>(part, f0, b.x, b.y);
        mma_16<BF>(part, f1, b.z, b.w);
      }
      if ((j + 1) % SPG == 0) {
        float s[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t word;
          asm volatile("ld.shared.u32 %0, [%1];" : "=r"(word) : "r"(wt + 1024 + 4 * ((j / SPG) * 16 + g + 8 * h)) : "memory");
          const int n = min((rb0 + rb) * 16 + g + 8 * h, a.N - 1);
          const int k = min((kb0 + kb) * I4_KB + (j / SPG) * SPG * 32, a.K - 1);
          const uint16_t v = (uint16_t)(word >> (((((int64_t)n * ng) + k / a.group) & 1) * 16));
          s[h] = a.scale_bf16 ? __uint_as_float((uint32_t)v << 16) : __half2float(__ushort_as_half(v));
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          acc[e] = fmaf(s[e >> 1], part[e], acc[e]);
          part[e] = 0.0f;
        }
      }
    }
    __syncwarp();
    if (++kb == nk || u + 1 == u1) {
      if (from_start && kb == nk) emit_full(); else emit_piece(from_start ? 1 : 0);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = 0.0f;
      if (kb == nk) {
        kb = 0;
        ++rb;
        from_start = true;
      }
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();

  // Row blocks cut between warps: the piece of the warp that began it (slot 1), then the others'.
  const int warp_of_units = I4_NW;
  for (int i = tid; i < nrb * 128; i += I4_NT) {
    const int b = i >> 7, e = i & 127, first = b * nk, last = first + nk - 1;
    if (nk == 0) {
      if (ks > 1) sums[i] = 0.0f;
      continue;
    }
    // The warp of unit u is the largest w with units * w / NW <= u.
    int w0 = (int)(((int64_t)first * warp_of_units) / units), w1 = (int)(((int64_t)last * warp_of_units) / units);
    while (w0 + 1 < I4_NW && (int64_t)units * (w0 + 1) / I4_NW <= first) ++w0;
    while (w1 + 1 < I4_NW && (int64_t)units * (w1 + 1) / I4_NW <= last) ++w1;
    if (w0 == w1) continue;
    float v = piece[(w0 * 2 + 1) * 128 + e];
    for (int w = w0 + 1; w <= w1; ++w)
      if ((int64_t)units * (w + 1) / I4_NW > (int64_t)units * w / I4_NW) v += piece[w * 2 * 128 + e];
    const int n = (rb0 + b) * 16 + (e >> 3), r = e & 7;
    if (ks > 1) sums[i] = v;
    else if (r < rows && n < a.N) i4_store(a, row0 + r, n, v);
  }
  if (ks > 1) {
    cl.sync();
    for (int b = rank; b < nrb; b += ks) {
      for (int i = tid; i < 128; i += I4_NT) {
        float v = 0.0f;
        for (int q = 0; q < ks; ++q) v += *cl.map_shared_rank(sums + b * 128 + i, q);
        const int n = (rb0 + b) * 16 + (i >> 3), r = i & 7;
        if (r < rows && n < a.N) i4_store(a, row0 + r, n, v);
      }
    }
    cl.sync();  // no CTA leaves while its sums are read
  }
}

}  // namespace lss
