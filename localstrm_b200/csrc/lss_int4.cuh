// lss_int4.cuh — products of a few rows with a matrix of 4-bit weights and group scales.
#pragma once

#include "lss_common.cuh"

namespace lss {

constexpr int I4_NW = 16;          // warps per CTA
constexpr int I4_NT = I4_NW * 32;
constexpr int I4_ST = 3;           // stages of the copy ring per warp
constexpr int I4_ROWS = 8;         // rows of x that one pass takes
constexpr int I4_KB = 128;         // columns per unit
constexpr int I4_RB = 32;          // matrix rows per unit
constexpr int I4_SUMS = I4_RB * I4_ROWS;  // results of one row block

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
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The first product of a sum.
template <bool BF>
__device__ __forceinline__ void mma_16_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (BF)
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
  else
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}

// (w & mask) | bits in one instruction.
__device__ __forceinline__ uint32_t and_or(uint32_t w, uint32_t mask, uint32_t bits) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(w), "r"(mask), "r"(bits));
  return r;
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
      uint32_t u = and_or(w >> (4 * i), 0x000f000fu, 0x43004300u);
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
      uint32_t u = and_or(s, 0x000f000fu, 0x64006400u), v = and_or(s, 0x00f000f0u, 0x64006400u);
      const __half2 a = __hsub2(*reinterpret_cast<__half2*>(&u), off);
      const __half2 b = __hfma2(*reinterpret_cast<__half2*>(&v), six, off16);
      r[2 * i] = *reinterpret_cast<const uint32_t*>(&a);
      r[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&b);
    }
  }
}

// Copies 16 bytes of which `valid` are read, the rest zero.
__device__ __forceinline__ void cp_async16z(uint32_t dst, const void* src, int valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid) : "memory");
}

// Where the 16 bytes `q` (32 columns) of row `r` of a unit lie: pieces permuted so that the rows that
// one shared load of 4, 8 or 16 bytes per lane serves at a time fall into different bank groups.
__device__ __forceinline__ uint32_t i4_offset(int r, int q) {
  const int line = r >> 1, swap = ((line & 1) << 1) | ((line >> 1) & 1);
  return (uint32_t)(line * 128 + (r & 1) * 64 + ((q ^ swap) << 4));
}

__device__ __forceinline__ void i4_store(const Int4Args& a, int row, int n, float v) {
  const int64_t at = (int64_t)row * a.y_stride + n;
  if (a.y_dtype == LSS_DTYPE_F32) reinterpret_cast<float*>(a.y)[at] = v;
  else if (a.y_dtype == LSS_DTYPE_BF16) reinterpret_cast<__nv_bfloat16*>(a.y)[at] = __float2bfloat16_rn(v);
  else reinterpret_cast<__half*>(a.y)[at] = __float2half_rn(v);
}

// Eight values of x (row r, columns k .. k + 7) as operand words in the order of int4_unpack's pairs; zero
// where `in` is false.  f32 values become P = 3 planes of bf16 that add up to them exactly (8 + 8 + 8
// bits, truncated).
template <int DT, int P>
__device__ __forceinline__ void i4_octet(const Int4Args& a, int r, int k, bool in, uint32_t (&out)[P][4]) {
  constexpr int ord[8] = {0, 4, 1, 5, 2, 6, 3, 7};
  const int64_t at = (int64_t)r * a.x_stride + k;
  if constexpr (DT == LSS_DTYPE_F32) {
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = in ? reinterpret_cast<const float*>(a.x)[at + e] : 0.0f;
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
#pragma unroll
      for (int e = 0; e < 4; ++e) out[p][e] = (uint32_t)h[ord[2 * e]] | ((uint32_t)h[ord[2 * e + 1]] << 16);
    }
  } else {
    uint16_t h[8];
    const uint16_t* src = reinterpret_cast<const uint16_t*>(a.x) + at;
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = 0;
    if (in) {  // K is a multiple of 32
      if (a.x_aligned) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(src));
        const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] = (uint16_t)(u[e >> 1] >> ((e & 1) * 16));
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] = src[e];
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) out[0][e] = (uint32_t)h[ord[2 * e]] | ((uint32_t)h[ord[2 * e + 1]] << 16);
  }
}

// Stages columns [k0, k0 + kn) of `rows` rows of x in shared memory as matrix operands.  The 8 columns
// that lane c of a row multiplies in step j of a unit (a 32-bit word of codes) are number
// 4 SPG (j / SPG) + SPG c + j % SPG of the unit's 16: a lane's words of one group are neighbours, and a
// step stays inside a group.  They lie at [plane][unit][j][row][c], 16 bytes each.
template <int DT, int SPG>
__device__ __forceinline__ void i4_stage_x(const Int4Args& a, int row0, int rows, int k0, int kn, unsigned char* xs) {
  constexpr int P = DT == LSS_DTYPE_F32 ? 3 : 1;
  const int groups = kn >> 3;  // kn is a multiple of 128; columns from K on are zero
  const int plane = (kn >> 5) * rows * 64;
  for (int i = threadIdx.x; i < rows * groups; i += blockDim.x) {
    const int r = i / groups, q = i - r * groups, k = k0 + q * 8;
    const int o = q & 15, gq = o / (4 * SPG), c = (o % (4 * SPG)) / SPG, j = gq * SPG + o % SPG;
    unsigned char* dst = xs + (((q >> 4) * 4 + j) * rows + r) * 64 + c * 16;
    uint32_t out[P][4];
    i4_octet<DT, P>(a, row0 + r, k, k < a.K, out);
#pragma unroll
    for (int p = 0; p < P; ++p) *reinterpret_cast<uint4*>(dst + p * plane) = make_uint4(out[p][0], out[p][1], out[p][2], out[p][3]);
  }
}

// y[r, n] = sum_g scale[n, g] * sum_{k in g} x[r, k] (code[n, k] - 8)  for up to 8 rows of x.
//
// A unit is 32 matrix rows times 128 columns (2 KB of codes).  A cluster of ks CTAs takes a range of
// 32-row blocks, each of its CTAs a slice of the columns; inside a CTA the units, row block by row
// block, are cut into equal ranges, one per warp, so that the bytes are spread evenly whatever N and K
// are.  Every warp streams its units through its own ring of asynchronous copies; x lies in shared
// memory as matrix operands for the whole kernel.  The codes are widened to exact 16-bit values of
// x's type (bf16 for f32 x, as three exact parts) and multiplied as the 16-row operand of
// mma.m16n8k16 with f32 sums; the group's sum is then scaled in f32.  Pieces of a row block that was
// cut between warps are added up in shared memory, those between CTAs through distributed shared
// memory, always in the same order.
// The bytes (0.5 per weight plus the scales) are what it cannot do without; what bounds it is the issue of
// instructions, about 360 per unit and warp, half of them the widening (11 per 8 weights in bf16, 9 in f16;
// the integer pipe takes 7 and 5 of those at two warps a cycle).  Units of 32 rows instead of 16 share a load
// of x and the loop's bookkeeping: 102 -> 82 us.
// Measured, 151,936 x 4096, groups of 128: one row 82 us in bf16 (3.9 TB/s, 0.61 of the copy rate; 86 to 96 us with the
// L2 cache swept between calls), 76 us in f16, 114 us in f32 (four rows 125); eight rows of bf16 86 us.
template <int DT, int SPG>  // SPG: 32-column steps per group (1, 2, or 4 for groups of 128 and more)
__global__ void __launch_bounds__(I4_NT, 1) lss_int4_kernel(Int4Args a, int row0, int rows, int ks) {
  constexpr bool BF = DT != LSS_DTYPE_F16;
  constexpr int P = DT == LSS_DTYPE_F32 ? 3 : 1;
  constexpr int SPU = 4 / SPG;  // scales per row and unit
  constexpr int NH = I4_RB / 8; // rows of a unit that a lane copies, and whose scales it holds
  constexpr uint32_t STAGE = I4_RB * I4_KB / 2;
  extern __shared__ __align__(128) unsigned char i4_sm[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
  cg::cluster_group cl = cg::this_cluster();
  const int rank = ks > 1 ? (int)cl.block_rank() : 0;
  const int cluster = blockIdx.x / ks, nclusters = gridDim.x / ks;
  const int NB = (a.N + I4_RB - 1) / I4_RB, KB = (a.K + I4_KB - 1) / I4_KB, ng = a.K / a.group;
  const int rb0 = (int)((int64_t)NB * cluster / nclusters), rb1 = (int)((int64_t)NB * (cluster + 1) / nclusters);
  const int kb0 = KB * rank / ks, kb1 = KB * (rank + 1) / ks, nk = kb1 - kb0;
  const int nrb = rb1 - rb0, units = nrb * nk;

  // Shared memory: rings, then the pieces (two per warp, 32 x 8 sums each), then the row blocks'
  // sums (clusters only), then x.
  const uint32_t ring = saddr(i4_sm) + (uint32_t)warp * (I4_ST * STAGE);
  float* piece = reinterpret_cast<float*>(i4_sm + I4_NW * I4_ST * STAGE);
  float* sums = piece + I4_NW * 2 * I4_SUMS;
  unsigned char* xs = reinterpret_cast<unsigned char*>(sums + (ks > 1 ? ((NB + nclusters - 1) / nclusters) * I4_SUMS : 0));

  const int u0 = (int)((int64_t)units * warp / I4_NW), u1 = (int)((int64_t)units * (warp + 1) / I4_NW);
  const int urb = u0 / nk, ukb = u0 - urb * nk;

  // Fetching side: the lane's 16-byte pieces of a unit, rows lane / 4 and every 8th one on, columns
  // 32 (lane % 4) on; 32-bit offsets into the CTA's rows.
  int iu = u0, irb = urb, ikb = ukb;
  const uint8_t* codes = a.packed + (int64_t)rb0 * I4_RB * (a.K >> 1);
  uint32_t src[NH], to[NH];
  const bool tail = a.K % I4_KB != 0;
  const bool tail_out = (KB - 1) * I4_KB + c * 32 >= a.K;  // the lane's columns of the last unit lie behind K
  auto aim = [&]() {
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      const int n = min(irb * I4_RB + g + 8 * h, a.N - 1 - rb0 * I4_RB);
      src[h] = (uint32_t)n * (uint32_t)(a.K >> 1) + (uint32_t)((kb0 + ikb) * (I4_KB / 2) + c * 16);
    }
  };
  aim();
#pragma unroll
  for (int h = 0; h < NH; ++h) to[h] = ring + i4_offset(g + 8 * h, c);
  auto issue = [&](uint32_t at) {
    if (iu < u1) {
      if (tail && kb0 + ikb == KB - 1) {
#pragma unroll
        for (int h = 0; h < NH; ++h) cp_async16z(to[h] + at, codes + (tail_out ? 0u : src[h]), tail_out ? 0 : 16);
      } else {
#pragma unroll
        for (int h = 0; h < NH; ++h) {
          cp_async16(to[h] + at, codes + src[h]);
          src[h] += I4_KB / 2;
        }
      }
      ++iu;
      if (++ikb == nk) {
        ikb = 0;
        ++irb;
        aim();
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int s = 0; s < I4_ST - 1; ++s) issue(s * STAGE);

  // Scales of rows g and every 8th one on, one unit ahead in registers.
  int srb = urb, skb = ukb, su = u0;
  const uint16_t* scales = a.scales + (int64_t)rb0 * I4_RB * ng;
  uint32_t sp[NH];
  uint16_t ahead[NH][SPU];
  const int gsteps = SPG == 4 ? a.group / I4_KB : 1;  // units per group
  int gleft = 0;
  auto aim_scales = [&]() {
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      const int n = min(srb * I4_RB + g + 8 * h, a.N - 1 - rb0 * I4_RB);
      sp[h] = (uint32_t)n * (uint32_t)ng + (uint32_t)(SPG == 4 ? (kb0 + skb) / gsteps : (kb0 + skb) * SPU);
    }
    gleft = SPG == 4 ? gsteps - (kb0 + skb) % gsteps : 1;
  };
  aim_scales();
  auto fetch_scales = [&]() {
    if (su < u1) {
      const int have = SPG == 4 ? 1 : min(SPU, ng - (kb0 + skb) * SPU);  // K may end inside the unit
#pragma unroll
      for (int h = 0; h < NH; ++h)
#pragma unroll
        for (int q = 0; q < SPU; ++q) ahead[h][q] = SPG == 4 || q < have ? __ldg(scales + sp[h] + q) : (uint16_t)0;
      const bool next = SPG < 4 || --gleft == 0;
      if (next) {
        gleft = gsteps;
#pragma unroll
        for (int h = 0; h < NH; ++h) sp[h] += SPU;
      }
      ++su;
      if (++skb == nk) {
        skb = 0;
        ++srb;
        aim_scales();
      }
    }
  };
  fetch_scales();
  i4_stage_x<DT, SPG>(a, row0, rows, kb0 * I4_KB, nk * I4_KB, xs);
  __syncthreads();

  constexpr int MT = I4_RB / 16;
  float acc[MT][4] = {};
  int rb = urb, kb = ukb;
  bool from_start = kb == 0;
  uint32_t stage = 0, fill = (I4_ST - 1) * STAGE;
  uint32_t from[NH];
#pragma unroll
  for (int h = 0; h < NH; ++h) from[h] = i4_offset(g + 8 * h, c * SPG >> 2) + ((c * SPG) & 3) * 4;
  // Lanes of rows that x does not have read its last one: their results are not stored.
  const uint32_t xbase = saddr(xs) + (uint32_t)(min(g, rows - 1) * 64 + c * 16), xstep = (uint32_t)rows * 64, xplane = (uint32_t)nk * 4 * xstep;
  uint32_t xat = xbase + (uint32_t)kb * 4 * xstep;
  auto emit_full = [&]() {
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int n = 16 * t + g + 8 * (e >> 1), r = 2 * c + (e & 1);
        if (ks > 1) {
          sums[rb * I4_SUMS + n * I4_ROWS + r] = acc[t][e];
        } else if (r < rows && (rb0 + rb) * I4_RB + n < a.N) {
          i4_store(a, row0 + r, (rb0 + rb) * I4_RB + n, acc[t][e]);
        }
      }
  };
  auto emit_piece = [&](int slot) {
    float* p = piece + (warp * 2 + slot) * I4_SUMS;
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) p[(16 * t + g + 8 * (e >> 1)) * I4_ROWS + 2 * c + (e & 1)] = acc[t][e];
  };
  for (int u = u0; u < u1; ++u) {
    cp_async_wait_group<I4_ST - 2>();
    __syncwarp();
    issue(fill);
    fill = fill + STAGE == I4_ST * STAGE ? 0 : fill + STAGE;
    float sc[NH][SPU];
    if (a.scale_bf16) {
#pragma unroll
      for (int h = 0; h < NH; ++h)
#pragma unroll
        for (int q = 0; q < SPU; ++q) sc[h][q] = __uint_as_float((uint32_t)ahead[h][q] << 16);
    } else {
#pragma unroll
      for (int h = 0; h < NH; ++h)
#pragma unroll
        for (int q = 0; q < SPU; ++q) sc[h][q] = __half2float(__ushort_as_half(ahead[h][q]));
    }
    fetch_scales();
    // The lane's words: SPG neighbours of each group; a group's first piece differs from the unit's
    // first by whole 16-byte pieces, which the permutation moves by exclusive or.
    uint32_t w[NH][4];
    const uint32_t at = ring + stage;
#pragma unroll
    for (int h = 0; h < NH; ++h)
#pragma unroll
      for (int q = 0; q < SPU; ++q) {
        const uint32_t p = at + (from[h] ^ (uint32_t)(q * SPG << 4));
        if constexpr (SPG == 4)
          asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[h][0]), "=r"(w[h][1]), "=r"(w[h][2]), "=r"(w[h][3]) : "r"(p) : "memory");
        else if constexpr (SPG == 2)
          asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[h][2 * q]), "=r"(w[h][2 * q + 1]) : "r"(p) : "memory");
        else
          asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[h][q]) : "r"(p) : "memory");
      }
    stage = stage + STAGE == I4_ST * STAGE ? 0 : stage + STAGE;
    float part[MT][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint4 b[P];
#pragma unroll
      for (int p = 0; p < P; ++p)
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(b[p].x), "=r"(b[p].y), "=r"(b[p].z), "=r"(b[p].w) : "r"(xat + p * xplane) : "memory");
      xat += xstep;
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        uint32_t lo[4], hi[4];
        int4_unpack<BF>(w[2 * t][j], lo);
        int4_unpack<BF>(w[2 * t + 1][j], hi);
        const uint32_t f0[4] = {lo[0], hi[0], lo[1], hi[1]}, f1[4] = {lo[2], hi[2], lo[3], hi[3]};
#pragma unroll
        for (int p = 0; p < P; ++p) {
          if (j % SPG == 0 && p == 0) mma_16_first<BF>(part[t], f0, b[p].x, b[p].y);
          else mma_16<BF>(part[t], f0, b[p].x, b[p].y);
          mma_16<BF>(part[t], f1, b[p].z, b[p].w);
        }
        if ((j + 1) % SPG == 0) {
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[t][e] = fmaf(sc[2 * t + (e >> 1)][j / SPG], part[t][e], acc[t][e]);
        }
      }
    }
    if (++kb == nk || u + 1 == u1) {
      if (from_start && kb == nk) emit_full(); else emit_piece(from_start ? 1 : 0);
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[t][e] = 0.0f;
      if (kb == nk) {
        kb = 0;
        xat = xbase;
        ++rb;
        from_start = true;
      }
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();

  // Row blocks cut between warps: the piece of the warp that began it (slot 1), then the others'.
  for (int i = tid; i < nrb * I4_SUMS; i += I4_NT) {
    const int b = i / I4_SUMS, e = i % I4_SUMS, first = b * nk, last = first + nk - 1;
    // The warp of unit u is the largest w with units * w / NW <= u.
    int w0 = (int)(((int64_t)first * I4_NW) / units), w1 = (int)(((int64_t)last * I4_NW) / units);
    while (w0 + 1 < I4_NW && (int64_t)units * (w0 + 1) / I4_NW <= first) ++w0;
    while (w1 + 1 < I4_NW && (int64_t)units * (w1 + 1) / I4_NW <= last) ++w1;
    if (w0 == w1) continue;
    float v = piece[(w0 * 2 + 1) * I4_SUMS + e];
    for (int w = w0 + 1; w <= w1; ++w)
      if ((int64_t)units * (w + 1) / I4_NW > (int64_t)units * w / I4_NW) v += piece[w * 2 * I4_SUMS + e];
    const int n = (rb0 + b) * I4_RB + e / I4_ROWS, r = e % I4_ROWS;
    if (ks > 1) sums[i] = v;
    else if (r < rows && n < a.N) i4_store(a, row0 + r, n, v);
  }
  if (ks > 1) {
    cl.sync();
    // The cluster's CTAs share the results out.
    for (int i = rank * I4_NT + tid; i < nrb * I4_SUMS; i += ks * I4_NT) {
      float v = 0.0f;
      for (int q = 0; q < ks; ++q) v += *cl.map_shared_rank(sums + i, q);
      const int n = rb0 * I4_RB + i / I4_ROWS, r = i % I4_ROWS;
      if (r < rows && n < a.N) i4_store(a, row0 + r, n, v);
    }
    cl.sync();  // no CTA leaves while its sums are read
  }
}

}  // namespace lss
