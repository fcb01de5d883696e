// lss_int4_tc.cuh — products of 9 to 64 rows with a matrix of 4-bit weights and group scales, on the
// fifth-generation tensor cores (tcgen05, operands and sums in tensor memory).
#pragma once

#include "lss_int4.cuh"

namespace lss {

constexpr int T4_NW = 16;              // warps: four teams of four
constexpr int T4_TEAMS = 4;
constexpr int T4_NT = T4_NW * 32;
constexpr int T4_ST = 3;               // stages of a warp's ring of codes (32 rows x 128 columns, 2 KB)
constexpr int T4_RB = 128;             // matrix rows of a team
constexpr long long T4_WAIT = 2000000000LL;  // about a second

struct Int4TcArgs {
  Int4Args a;
  const unsigned char* xop;  // x as matrix operand, see lss_int4_operand_kernel
  float* part;               // [ks][rows][N - first] sums of the column slices (ks > 1)
  int row0, rows, ks, full, rest;  // row blocks per CTA, one per team: T4_TEAMS in the first `full`, `rest` in the others
  int first;                 // first matrix row of the others, which have ks column slices each
};

__device__ __forceinline__ void tc_alloc(uint32_t* out, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(saddr(out)), "r"(cols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tc_free(uint32_t base, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols) : "memory");
}
__device__ __forceinline__ void tc_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// 16 words per lane to 16 columns of the warp's 32 lanes.
__device__ __forceinline__ void tc_st16(uint32_t at, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tc_ld16(uint32_t at, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(at)
      : "memory");
}
// D (+)= A B with A in tensor memory and B in shared memory; one thread issues it.
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, bool add) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 b;\n mov.b64 b, {%2, %3};\n setp.ne.b32 p, %5, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n}\n" ::"r"(d),
      "r"(a), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"((uint32_t)add)
      : "memory");
}
// True for one thread of a warp whose lanes are all here.  Products are issued under it, by a warp that
// otherwise stays together, so that their operands are known to be the same for all lanes: under
// `lane == 0` every tcgen05.mma took 60 to 125 cycles to issue.
__device__ __forceinline__ bool tc_elect() {
  uint32_t one;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(one));
  return one != 0;
}
// Arrives on `bar` when the products issued so far by this thread are done.
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(saddr(bar)) : "memory");
}
// Shared-memory operand whose rows are 128-byte lines (64 16-bit columns) in 8-line groups, pieces of
// 16 bytes permuted inside a line by the line number (the 128-byte swizzle): the two halves of its
// descriptor.  The lower one counts the address in 16 bytes.
__device__ __forceinline__ uint32_t tc_desc_lo(uint32_t addr) { return ((addr >> 4) & 0x3fffu) | (1u << 16); }
constexpr uint32_t TC_DESC_HI = (1024u >> 4) | (1u << 14) | (2u << 29);
// 16-bit operands, f32 sums, both operands along columns; M = 128.
__device__ __forceinline__ constexpr uint32_t tc_idesc(bool bf16, int n) {
  return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}
// Bounded wait; once one has given up anywhere in the CTA, all others give up at once.  The thread
// sleeps until the phase completes (asking again and again would take the widening's issue slots).
__device__ __forceinline__ bool tc_wait(uint64_t* bar, uint32_t parity, volatile int* failed) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  for (;;) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(saddr(bar)), "r"(parity), "r"(100000u)
        : "memory");
    if (ok) return true;
    if (*failed) return false;
    if (clock64() - t0 > T4_WAIT) {
      *failed = 1;
      return false;
    }
  }
}

// Writes x as the operand that the product kernel copies: [unit of 128 columns][plane][half][NR rows][128
// bytes], 16-byte pieces in the order of int4_unpack's pairs and permuted by row (tc_desc_lo); zero
// behind the last row and column.  f32 values become three bf16 planes that add up to them.
template <int DT, int NR>
__global__ void __launch_bounds__(256) lss_int4_operand_kernel(Int4Args a, int row0, int rows, unsigned char* xop) {
  constexpr int P = DT == LSS_DTYPE_F32 ? 3 : 1;
  pdl_trigger();
  const int KB = (a.K + I4_KB - 1) / I4_KB;
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= KB * NR * 16) return;
  const int o = i & 15, r = (i >> 4) % NR, u = (i >> 4) / NR, k = u * I4_KB + o * 8;
  uint32_t out[P][4];
  i4_octet<DT, P>(a, row0 + r, k, r < rows && k < a.K, out);
  unsigned char* dst = xop + ((size_t)u * P * 2 + (o >> 3)) * NR * 128 + r * 128 + (((o & 7) ^ (r & 7)) << 4);
#pragma unroll
  for (int p = 0; p < P; ++p) *reinterpret_cast<uint4*>(dst + (size_t)p * 2 * NR * 128) = make_uint4(out[p][0], out[p][1], out[p][2], out[p][3]);
}

// The product of lss_int4_kernel for NR = 16, 32 or 64 rows of x.
//
// A team of four warps has 128 matrix rows, one per thread and lane of tensor memory: each thread
// widens its row's 128 codes of a unit (64 bytes) to exact 16-bit values and stores them as the
// 128 x 128 left operand in tensor memory; the right one is the unit's x in shared memory, fetched by one
// bulk copy per unit for all teams.  One thread issues the 8 products (x 3 planes for f32 x) of the
// unit into a sum of its own per group; when they are done every thread reads its row's NR sums back,
// scales them in f32 and adds them up in registers.  The codes never go to shared memory as 16-bit
// values, whose bandwidth (128 B per cycle and SM) could not carry them at the rate of HBM.  The teams drift
// apart by up to XS - 1 units, so that the widening of one overlaps the products of another.
// Measured, 128,256 x 4096, groups of 128, bf16: 64 rows 109 us (122 with the L2 cache swept between calls), 16 rows
// 86 us (lss_int4_kernel eight rows at a time: 591 and 164 us).  f32 x, three products per unit, cache swept: 16 rows 104 us,
// 32 rows 128, 64 rows 190.  More than 64 rows repeat all of it (151,936 x 4096, bf16: 128 rows 264 us, 256 rows 520).  Bound by the instructions of the widening, as there, and by the chain of a unit (codes,
// widening, products, sums), which four teams a CTA hide in part.
// Tensor memory: 64 columns of left operand and 64 of sums per team, all 512.
// A range of columns per CTA (ks of them) where there are few row blocks, or few behind the last full wave;
// lss_int4_sum_kernel adds up.
template <int DT, int SPG, int NR>
__global__ void __launch_bounds__(T4_NT, 1) lss_int4_tc_kernel(Int4TcArgs t) {
  constexpr bool BF = DT != LSS_DTYPE_F16;
  constexpr int P = DT == LSS_DTYPE_F32 ? 3 : 1;
  constexpr int SPU = 4 / SPG;                               // groups per unit
  constexpr int GR = 64 / NR < SPU ? 64 / NR : SPU;          // groups whose sums fit side by side
  constexpr int XB = P * NR * 256;                           // bytes of a unit's x
  constexpr int XS = P == 1 ? 4 : 2;
  constexpr uint32_t STAGE = 32 * I4_KB / 2;
  extern __shared__ __align__(1024) unsigned char t4_sm[];
  __shared__ __align__(8) uint64_t xfull[XS], xempty[XS], done[T4_TEAMS];
  __shared__ uint32_t tmem_base;
  __shared__ int failed;
  const Int4Args& a = t.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, team = warp >> 2, quarter = warp & 3;
  const int NB = (a.N + T4_RB - 1) / T4_RB, KB = (a.K + I4_KB - 1) / I4_KB, ng = a.K / a.group;
  const int ks = (int)blockIdx.x < t.full ? 1 : t.ks, behind = (int)blockIdx.x - t.full;
  const int slice = ks > 1 ? behind % ks : 0, cta = ks > 1 ? t.full + behind / ks : (int)blockIdx.x;
  const int block0 = cta < t.full ? cta * T4_TEAMS : t.full * T4_TEAMS + (cta - t.full) * t.rest;
  const int active = min(cta < t.full ? T4_TEAMS : t.rest, NB - block0);  // teams with work
  const int kb0 = (int)((int64_t)KB * slice / ks), nu = (int)((int64_t)KB * (slice + 1) / ks) - kb0;
  // 1024-byte alignment of the operand within the dynamic part
  unsigned char* xs = t4_sm + ((1024 - (saddr(t4_sm) & 1023)) & 1023);
  const uint32_t ring = saddr(xs) + XS * XB + (uint32_t)warp * (T4_ST * STAGE);

  if (warp == 0) tc_alloc(&tmem_base, 512);
  if (tid == 0) {
    failed = 0;
    for (int i = 0; i < XS; ++i) {
      mbar_init(&xfull[i], 1);
      mbar_init(&xempty[i], active);
    }
    for (int i = 0; i < T4_TEAMS; ++i) mbar_init(&done[i], 1);
    fence_barrier_init();
  }

  // Codes: rows lane / 4 and every 8th one on of the warp's 32, columns 32 (lane % 4) on.
  const int g = lane >> 2, c = lane & 3;
  const int n0 = (block0 + team) * T4_RB + quarter * 32;     // first matrix row of the warp
  const bool works = team < active;
  uint32_t src[4], to[4];
  const uint8_t* codes = a.packed + (int64_t)min(n0, a.N - 1) * (a.K >> 1);
  const bool tail = a.K % I4_KB != 0, tail_out = (KB - 1) * I4_KB + c * 32 >= a.K;
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    const int n = min(n0 + g + 8 * h, a.N - 1) - min(n0, a.N - 1);
    src[h] = (uint32_t)n * (uint32_t)(a.K >> 1) + (uint32_t)(kb0 * (I4_KB / 2) + c * 16);
    to[h] = ring + i4_offset(g + 8 * h, c);
  }
  int iu = 0;
  auto issue = [&](uint32_t at) {
    if (iu < nu) {
      if (tail && kb0 + iu == KB - 1) {
#pragma unroll
        for (int h = 0; h < 4; ++h) cp_async16z(to[h] + at, codes + (tail_out ? 0u : src[h]), tail_out ? 0 : 16);
      } else {
#pragma unroll
        for (int h = 0; h < 4; ++h) cp_async16(to[h] + at, codes + src[h]);
      }
#pragma unroll
      for (int h = 0; h < 4; ++h) src[h] += I4_KB / 2;
      ++iu;
    }
    cp_async_commit();
  };
  if (works) {
#pragma unroll
    for (int s = 0; s < T4_ST - 1; ++s) issue(s * STAGE);
  }
  // Scales of the thread's row, one unit ahead.
  const uint16_t* sp = a.scales + (int64_t)min(n0 + lane, a.N - 1) * ng;
  uint16_t ahead[SPU];
  const int gsteps = SPG == 4 ? a.group / I4_KB : 1;
  auto fetch_scales = [&](int u) {
    const int k = kb0 + u;
    if (SPG == 4) {
      ahead[0] = __ldg(sp + (gsteps == 1 ? k : k / gsteps));
    } else {
#pragma unroll
      for (int q = 0; q < SPU; ++q) ahead[q] = k * SPU + q < ng ? __ldg(sp + k * SPU + q) : (uint16_t)0;
    }
  };
  fetch_scales(0);
  tc_before_sync();
  __syncthreads();
  tc_after_sync();
  const uint32_t tmem = tmem_base;

  pdl_wait();  // x's operand form comes from the kernel before
  auto fetch_x = [&](int u) {
    const int b = u % XS;
    mbar_expect_tx(&xfull[b], XB);
    bulk_g2s(xs + b * XB, t.xop + (size_t)(kb0 + u) * XB, XB, &xfull[b]);
  };
  // Unit u's copy waits for unit u - XS of all teams; the thread that issues it asks one unit late, so that its
  // own team is not held up by the slowest one.
  int xu = 0;
  const bool fetches = tid == 96;  // team 0's last warp: its first one issues products
  if (fetches)
    for (; xu < min(XS, nu); ++xu) fetch_x(xu);

  float acc[NR];
#pragma unroll
  for (int i = 0; i < NR; ++i) acc[i] = 0.0f;
  const uint32_t a_at = tmem + team * 128, d_at = a_at + 64, lanes = (uint32_t)(quarter * 32) << 16;
  constexpr uint32_t idesc = tc_idesc(BF, NR);
  if (works) {
    uint32_t stage = 0, fill = (T4_ST - 1) * STAGE, phase = 0;
    for (int u = 0; u < nu; ++u) {
      const int b = u % XS;
      cp_async_wait_group<T4_ST - 2>();
      __syncwarp();
      issue(fill);
      fill = fill + STAGE == T4_ST * STAGE ? 0 : fill + STAGE;
      float sc[SPU];
      if (a.scale_bf16) {
#pragma unroll
        for (int q = 0; q < SPU; ++q) sc[q] = __uint_as_float((uint32_t)ahead[q] << 16);
      } else {
#pragma unroll
        for (int q = 0; q < SPU; ++q) sc[q] = __half2float(__ushort_as_half(ahead[q]));
      }
      if (u + 1 < nu) fetch_scales(u + 1);
      const uint32_t at = ring + stage + i4_offset(lane, 0);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        uint32_t w[4], r[16];
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at ^ (uint32_t)(q << 4)) : "memory");
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t v[4];
          int4_unpack<BF>(w[j], v);
#pragma unroll
          for (int e = 0; e < 4; ++e) r[4 * j + e] = v[e];
        }
        tc_st16(a_at + lanes + 16 * q, r);
      }
      stage = stage + STAGE == T4_ST * STAGE ? 0 : stage + STAGE;
      tc_wait_st();
#pragma unroll
      for (int g0 = 0; g0 < SPU; g0 += GR) {
        tc_before_sync();
        asm volatile("bar.sync %0, 128;" ::"r"(1 + team) : "memory");
        if (quarter == 0) {
          tc_after_sync();
          if (g0 == 0) tc_wait(&xfull[b], (u / XS) & 1, &failed);
          __syncwarp();
          if (tc_elect() && !*(volatile int*)&failed) {
            const uint32_t x0 = tc_desc_lo(saddr(xs) + b * XB);
#pragma unroll
            for (int s = g0 * 2 * SPG; s < (g0 + GR) * 2 * SPG; ++s)
#pragma unroll
              for (int p = 0; p < P; ++p)
                tc_mma_ts(d_at + (s / (2 * SPG) - g0) * NR, a_at + 8 * s, x0 + ((p * 2 + (s >> 2)) * NR * 128 + (s & 3) * 32) / 16, TC_DESC_HI,
                          idesc, s % (2 * SPG) != 0 || p > 0);
            tc_commit(&done[team]);
            if (g0 + GR >= SPU) tc_commit(&xempty[b]);
          }
        }
        tc_wait(&done[team], phase, &failed);
        phase ^= 1;
        tc_after_sync();
#pragma unroll
        for (int q = 0; q < GR; ++q)
#pragma unroll
          for (int i = 0; i < NR; i += 16) {
            uint32_t d[16];
            tc_ld16(d_at + lanes + q * NR + i, d);
            tc_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i + e] = fmaf(sc[g0 + q], __uint_as_float(d[e]), acc[i + e]);
          }
      }
      if (fetches && u > 0 && xu < nu) {  // the place of unit u - 1
        if (tc_wait(&xempty[xu % XS], ((xu / XS) - 1) & 1, &failed)) fetch_x(xu);
        ++xu;
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    const int n = n0 + lane;
    if (n < a.N) {
      const bool bad = *(volatile int*)&failed;  // a wait gave up: the results say so
#pragma unroll
      for (int i = 0; i < NR; ++i)
        if (i < t.rows) {
          const float v = bad ? __int_as_float(0x7fffffff) : acc[i];
          if (ks > 1) t.part[((size_t)slice * t.rows + i) * (a.N - t.first) + n - t.first] = v;
          else i4_store(a, t.row0 + i, n, v);
        }
    }
  }
  tc_before_sync();
  __syncthreads();
  tc_after_sync();
  if (*(volatile int*)&failed) {  // copies and products may still run: they get a quarter of a second
    const long long t0 = clock64();
    while (clock64() - t0 < T4_WAIT / 4) __nanosleep(1000);
    __syncthreads();
  }
  if (warp == 0) tc_free(tmem, 512);
}

// Adds up the column slices' sums, in order.
static __global__ void __launch_bounds__(256) lss_int4_sum_kernel(Int4TcArgs t) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, cols = t.a.N - t.first, size = t.rows * cols;
  if (i >= size) return;
  float v = 0.0f;
  for (int s = 0; s < t.ks; ++s) v += t.part[s * size + i];
  const int r = (int)(i / cols);
  i4_store(t.a, t.row0 + r, t.first + (int)(i - r * cols), v);
}

}  // namespace lss
