// lss_decode.cu — C ABI of the decode-step operators around the sampler: 4-bit products, block
// tables, the 8-bit key/value cache and its attention.
#include "lss_attend_host.cuh"
#include "lss_blocks.cuh"
#include "lss_int4_tc.cuh"
#include "lss_kvcache.cuh"

// ---------------------------------------------------------------- 4-bit products
static constexpr int I4_SMEM = 227 * 1024;

// Clusters of k CTAs with an SM's whole shared memory that run at a time: fewer than SMs / k, as a cluster lies in one
// group of SMs whose number need not be a multiple of k.  Asked once per device; without one, SMs / k.
static int cluster_count(int dev, int k, int sms) {
  static int n[MAX_DEV][4] = {};
  int& got = n[dev][log2_of(k)];
  std::lock_guard<std::mutex> lock(g_mu);
  if (got == 0) {
    auto* kern = lss_int4_kernel<LSS_DTYPE_BF16, 4>;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(k * sms), 1, 1);
    cfg.blockDim = dim3(I4_NT, 1, 1);
    cfg.dynamicSmemBytes = I4_SMEM;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)k;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    int c = 0;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, I4_SMEM) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&c, kern, &cfg) != cudaSuccess || c < 1) {
      cudaGetLastError();
      return std::max(1, sms / k);
    }
    got = c;
  }
  return got;
}

// Split of lss_int4_kernel: CTAs per row block range (ks), ranges, rows of x that a launch's shared memory takes (0:
// not even one in any split).  The matrix is read once per `most` rows: of the splits with the fewest passes the one
// with the fewest units in the fullest CTA; a cluster's exchange costs about as much as 8 units, and its row blocks'
// sums take 16 KB at most.  (Fewest units alone: 8 rows of 4096 x 14,336 in three passes, 60 us in bf16, and eight,
// 169 us in f32.)  There are no more ranges than clusters run at a time (one row of 14,336 x 4096 in SMs / 4 ranges:
// two waves, 37 us).
struct I4Plan {
  int ks, nclusters, sums, most;  // sums: bytes of the row blocks' sums
  int passes(int rows) const { return (rows + most - 1) / most; }
};
static constexpr int I4_FIXED = I4_NW * I4_ST * (I4_RB * I4_KB / 2) + I4_NW * 2 * I4_SUMS * 4;
static I4Plan i4_plan(int rows, int N, int K, int planes, int dev) {
  const int NB = (N + I4_RB - 1) / I4_RB, KB = (K + I4_KB - 1) / I4_KB, sms = sm_count(dev);
  I4Plan best{1, 0, 0, 0};
  int64_t best_cost = 0;
  for (int k = 1; k <= 8 && k <= KB; k <<= 1) {
    const int nc = std::min(NB, k == 1 ? sms : cluster_count(dev, k, sms)), nrb = (NB + nc - 1) / nc, units = (KB + k - 1) / k;
    if (k > 1 && nrb > 16) continue;
    const int sums = k > 1 ? nrb * I4_SUMS * 4 : 0;
    const int64_t most = (I4_SMEM - I4_FIXED - sums) / ((int64_t)units * I4_KB * 2 * planes);
    const int64_t cost = (int64_t)nrb * units + (k > 1 ? 8 : 0);
    if (most < 1) continue;
    const I4Plan p{k, nc, sums, (int)std::min((int64_t)I4_ROWS, most)};
    if (best.most == 0 || p.passes(rows) < best.passes(rows) || (p.passes(rows) == best.passes(rows) && cost < best_cost)) {
      best_cost = cost;
      best = p;
    }
  }
  return best;
}

template <int DT, int SPG>
static cudaError_t launch_int4(const Int4Args& a, const I4Plan& p, cudaStream_t st) {
  static SmemSet set;
  constexpr int planes = DT == LSS_DTYPE_F32 ? 3 : 1;
  const int KB = (a.K + I4_KB - 1) / I4_KB;
  for (int r0 = 0; r0 < a.rows; r0 += p.most) {
    const int rows = std::min(p.most, a.rows - r0);
    const int smem = I4_FIXED + p.sums + rows * ((KB + p.ks - 1) / p.ks) * I4_KB * 2 * planes;
    cudaError_t e = allow_smem(lss_int4_kernel<DT, SPG>, set, device_index(), smem);
    if (e != cudaSuccess) return e;
    e = launch(lss_int4_kernel<DT, SPG>, (unsigned)(p.nclusters * p.ks), I4_NT, smem, p.ks, false, st, a, r0, rows, p.ks);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

// Nine rows and more, and rows of x too long for shared memory: the tensor-memory kernel, 64 rows of x at a time.
struct TcPlan {
  int ctas, full, rest, ks, first;  // CTAs; the first `full` have T4_TEAMS row blocks, the others `rest` and a slice of
                                    // the columns; first matrix row of the others
  size_t xop, part;
};
// The row blocks behind the last full wave of T4_TEAMS per SM: a unit of 128 columns takes about 1 us and an eighth of
// one per team (its chain of codes, widening, products and sums is only in part hidden by the other teams), a CTA's
// start and end eight units, slices a second launch and 1 ns per 300 of their sums.  So few teams per CTA on all SMs (64 rows, 128,256
// x 4096: 120 -> 109 us), or more of them with a slice of the columns each (151,936 x 4096, three blocks behind two
// waves: 150 -> 128 us; 100,000 x 4096, 190 behind one: 104 -> 102 us, 14,336 x 4096: 45 -> 36), whichever is less.
static TcPlan tc_plan(int rows, int N, int K, int x_dtype, int sms) {
  TcPlan p;
  const int NB = (N + T4_RB - 1) / T4_RB, KB = (K + I4_KB - 1) / I4_KB;
  p.full = (NB - 1) / (T4_TEAMS * sms) * sms;
  const int left = NB - p.full * T4_TEAMS;
  int64_t best = INT64_MAX;
  for (int t = 1; t <= T4_TEAMS; ++t) {
    const int behind = (left + t - 1) / t;
    if (behind > sms) continue;
    const int units = (KB + std::min(KB, sms / behind) - 1) / std::min(KB, sms / behind), ks = (KB + units - 1) / units;
    // ns
    const int64_t cost = (int64_t)(units + 8) * (1000 + 125 * t) + (ks > 1 ? 2500 + (int64_t)ks * std::min(rows, 64) * left * T4_RB / 300 : 0);
    if (cost < best) {
      best = cost;
      p.rest = t;
      p.ks = ks;
      p.ctas = p.full + behind * ks;
    }
  }
  p.first = p.full * T4_TEAMS * T4_RB;
  const int most = std::min(rows, 64);
  p.xop = (size_t)KB * (x_dtype == LSS_DTYPE_F32 ? 3 : 1) * 64 * 256;
  p.part = p.ks > 1 ? (size_t)p.ks * most * (N - p.first) * sizeof(float) : 0;
  return p;
}

template <int DT, int SPG, int NR>
static cudaError_t launch_int4_tc(const Int4Args& a, int row0, int rows, const TcPlan& p, unsigned char* ws, cudaStream_t st) {
  static SmemSet set;
  constexpr int planes = DT == LSS_DTYPE_F32 ? 3 : 1;
  constexpr int smem = 1024 + (planes == 1 ? 4 : 2) * planes * NR * 256 + T4_NW * T4_ST * (32 * I4_KB / 2);
  cudaError_t e = allow_smem(lss_int4_tc_kernel<DT, SPG, NR>, set, device_index(), smem);
  if (e != cudaSuccess) return e;
  const int KB = (a.K + I4_KB - 1) / I4_KB;
  Int4TcArgs t{a, ws, reinterpret_cast<float*>(ws + p.xop), row0, rows, p.ks, p.full, p.rest, p.first};
  e = launch(lss_int4_operand_kernel<DT, NR>, (unsigned)((KB * NR * 16 + 255) / 256), 256, 0, 1, false, st, a, row0, rows, ws);
  if (e != cudaSuccess) return e;
  e = launch(lss_int4_tc_kernel<DT, SPG, NR>, (unsigned)p.ctas, T4_NT, smem, 1, true, st, t);
  if (e != cudaSuccess || p.ks == 1) return e;
  return launch(lss_int4_sum_kernel, (unsigned)(((int64_t)rows * (a.N - p.first) + 255) / 256), 256, 0, 1, false, st, t);
}

// Up to eight rows: lss_int4_kernel, unless it would need more than one pass and the workspace has room for the other
// one (or x does not fit at all, when the workspace has to).
template <int DT, int SPG>
static cudaError_t launch_int4_rows(const Int4Args& a, void* ws, size_t ws_bytes, cudaStream_t st) {
  const int dev = device_index(), sms = sm_count(dev);
  if (a.rows <= I4_ROWS) {
    const I4Plan p = i4_plan(a.rows, a.N, a.K, DT == LSS_DTYPE_F32 ? 3 : 1, dev);
    const TcPlan t = tc_plan(a.rows, a.N, a.K, DT, sms);
    const bool room = ws && aligned_to(ws, 16) && ws_bytes >= t.xop + t.part;
    if (p.most > 0 && (p.passes(a.rows) == 1 || !room)) return launch_int4<DT, SPG>(a, p, st);
  }
  const TcPlan p = tc_plan(a.rows, a.N, a.K, DT, sms);
  unsigned char* w = reinterpret_cast<unsigned char*>(ws);
  for (int r0 = 0; r0 < a.rows; r0 += 64) {
    const int rows = std::min(64, a.rows - r0);
    const cudaError_t e = rows <= 16   ? launch_int4_tc<DT, SPG, 16>(a, r0, rows, p, w, st)
                          : rows <= 32 ? launch_int4_tc<DT, SPG, 32>(a, r0, rows, p, w, st)
                                       : launch_int4_tc<DT, SPG, 64>(a, r0, rows, p, w, st);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

template <int DT>
static cudaError_t launch_int4_group(const Int4Args& a, void* ws, size_t ws_bytes, cudaStream_t st) {
  if (a.group == 32) return launch_int4_rows<DT, 1>(a, ws, ws_bytes, st);
  if (a.group == 64) return launch_int4_rows<DT, 2>(a, ws, ws_bytes, st);
  return launch_int4_rows<DT, 4>(a, ws, ws_bytes, st);
}

extern "C" {

size_t lss_int4_workspace_bytes(int rows, int K, int x_dtype, int N) {
  if (rows < 1 || K < 1 || N < 1) return 0;
  const int dev = device_index(), sms = sm_count(dev);
  if (rows <= I4_ROWS && i4_plan(rows, N, K, x_dtype == LSS_DTYPE_F32 ? 3 : 1, dev).most > 0) return 0;
  const TcPlan p = tc_plan(rows, N, K, x_dtype, sms);
  return p.xop + p.part;
}

size_t lss_int4_workspace_one_pass_bytes(int rows, int K, int x_dtype, int N) {
  if (rows < 1 || K < 1 || N < 1) return 0;
  const int dev = device_index(), sms = sm_count(dev);
  if (rows <= I4_ROWS) {
    const I4Plan p = i4_plan(rows, N, K, x_dtype == LSS_DTYPE_F32 ? 3 : 1, dev);
    if (p.most > 0 && p.passes(rows) == 1) return 0;
  }
  const TcPlan p = tc_plan(rows, N, K, x_dtype, sms);
  return p.xop + p.part;
}

int lss_int4_matvec(const void* x, int x_dtype, int rows, int K, int64_t x_stride, const uint8_t* packed,
                    const void* scales, int scale_dtype, int N, int group, void* y, int y_dtype,
                    int64_t y_stride, void* workspace, size_t workspace_bytes, void* stream) {
  if (rows < 0 || N < 1 || K < 32 || K % 32 != 0 || x_stride < K || y_stride < N) return LSS_ERR_INVALID_ARG;
  if (!known_dtype(x_dtype) || !known_dtype(y_dtype)) return LSS_ERR_INVALID_ARG;
  if (scale_dtype != LSS_DTYPE_BF16 && scale_dtype != LSS_DTYPE_F16) return LSS_ERR_INVALID_ARG;
  if ((group != 32 && group != 64 && (group < 128 || group % 128 != 0)) || K % group != 0) return LSS_ERR_INVALID_ARG;
  if (rows == 0) return LSS_OK;
  if (!x || !packed || !scales || !y || !aligned_to(packed, 16) || !aligned_to(scales, 2)) return LSS_ERR_INVALID_ARG;
  const size_t need = lss_int4_workspace_bytes(rows, K, x_dtype, N);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned_to(workspace, 16))) return LSS_ERR_WORKSPACE;
  const int64_t xe = x_dtype == LSS_DTYPE_F32 ? 4 : 2, ye = y_dtype == LSS_DTYPE_F32 ? 4 : 2;
  if (rows_overlap(x, x_stride * xe, K * xe, y, y_stride * ye, N * ye, rows)) return LSS_ERR_INVALID_ARG;
  Int4Args a{};
  a.x = x;
  a.x_stride = x_stride;
  a.rows = rows;
  a.K = K;
  a.N = N;
  a.packed = packed;
  a.scales = reinterpret_cast<const uint16_t*>(scales);
  a.group = group;
  a.scale_bf16 = scale_dtype == LSS_DTYPE_BF16;
  a.y = y;
  a.y_dtype = y_dtype;
  a.y_stride = y_stride;
  a.x_aligned = aligned_to(x, 16) && x_stride % 8 == 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e;
  switch (x_dtype) {
    case LSS_DTYPE_F32: e = launch_int4_group<LSS_DTYPE_F32>(a, workspace, workspace_bytes, st); break;
    case LSS_DTYPE_BF16: e = launch_int4_group<LSS_DTYPE_BF16>(a, workspace, workspace_bytes, st); break;
    default: e = launch_int4_group<LSS_DTYPE_F16>(a, workspace, workspace_bytes, st); break;
  }
  return status_of(e);
}

int lss_block_plan(int32_t* table, int64_t table_stride, int width, const int32_t* lens,
                   const int32_t* new_lens, int B, int block_size, const int32_t* free_blocks, int num_blocks,
                   const int32_t* n_free, int capacity, int64_t* slots, int32_t* positions, int32_t* starts,
                   int32_t* granted, int32_t* lens_out, int32_t* n_free_out, void* stream) {
  if (!table_ok(table, table_stride, width, B, block_size, num_blocks) || capacity < 0) return LSS_ERR_INVALID_ARG;
  if (B > LSS_BLOCK_MAX_ROWS) return LSS_ERR_UNSUPPORTED;
  if (!free_blocks || !n_free || !starts || !n_free_out) return LSS_ERR_INVALID_ARG;
  if (B > 0 && (!lens || !new_lens || !granted || !lens_out)) return LSS_ERR_INVALID_ARG;
  if (capacity > 0 && (!slots || !positions)) return LSS_ERR_INVALID_ARG;
  if (cut(lens_out, lens, B) || cut(lens_out, new_lens, B)) return LSS_ERR_INVALID_ARG;
  PlanArgs a{table, table_stride, width, lens, new_lens, B, block_size, num_blocks, capacity, free_blocks,
             n_free, slots, positions, starts, granted, lens_out, n_free_out};
  static SmemSet set;
  const int dev = device_index(), smem = 8 * B;
  if (smem > 40 * 1024) {
    const cudaError_t e = allow_smem(lss_plan_kernel, set, dev, smem);
    if (e != cudaSuccess) return status_of(e);
  }
  const int64_t want = ((int64_t)capacity + BL_NT - 1) / BL_NT;
  const bool in_place = n_free_out == n_free || lens_out == lens || lens_out == new_lens;
  const int ctas = in_place ? cluster_for(want, BL_MAXCL) : (int)std::max((int64_t)1, std::min(want, (int64_t)sm_count(dev)));
  return status_of(launch(lss_plan_kernel, (unsigned)ctas, BL_NT, (size_t)smem, in_place ? ctas : 1, false,
                          reinterpret_cast<cudaStream_t>(stream), a));
}

int lss_block_release(const int32_t* table, int64_t table_stride, int width, const int32_t* lens,
                      const int32_t* codes, int B, int block_size, int32_t* free_blocks, int num_blocks,
                      const int32_t* n_free, int32_t* lens_out, int32_t* n_free_out, void* stream) {
  if (!table_ok(table, table_stride, width, B, block_size, num_blocks)) return LSS_ERR_INVALID_ARG;
  if (B > LSS_BLOCK_MAX_ROWS) return LSS_ERR_UNSUPPORTED;
  if (!free_blocks || !n_free || !n_free_out) return LSS_ERR_INVALID_ARG;
  if (B > 0 && (!lens || !codes || !lens_out)) return LSS_ERR_INVALID_ARG;
  if (cut(lens_out, lens, B) || cut(lens_out, codes, B)) return LSS_ERR_INVALID_ARG;
  ReleaseArgs a{table, table_stride, width, lens, codes, B, block_size, num_blocks, free_blocks, n_free, lens_out, n_free_out};
  static SmemSet set;
  const int dev = device_index(), smem = 4 * B;
  if (smem > 40 * 1024) {
    const cudaError_t e = allow_smem(lss_release_kernel, set, dev, smem);
    if (e != cudaSuccess) return status_of(e);
  }
  const int ctas = cluster_for((B + 31) / 32, BL_MAXCL);
  return status_of(launch(lss_release_kernel, (unsigned)ctas, BL_NT, (size_t)smem, ctas, false,
                          reinterpret_cast<cudaStream_t>(stream), a));
}

int lss_kv_append(const void* k, int64_t k_token_stride, int64_t k_head_stride, const void* v,
                  int64_t v_token_stride, int64_t v_head_stride, int dtype, int T, int heads, int dim,
                  uint8_t* k_cache, uint8_t* v_cache, float* k_scale, float* v_scale, int num_blocks,
                  int block_size, const int32_t* table, int64_t table_stride, int width, const int32_t* starts,
                  const int32_t* granted, const int32_t* lens, int B, void* stream) {
  if (!known_dtype(dtype) || T < 0 || heads < 1 || dim < 8 || dim % 8 != 0 || !block_size_ok(block_size))
    return LSS_ERR_INVALID_ARG;
  if (k_token_stride < 0 || k_head_stride < 0 || v_token_stride < 0 || v_head_stride < 0) return LSS_ERR_INVALID_ARG;
  if (!table_ok(table, table_stride, width, B, block_size, num_blocks)) return LSS_ERR_INVALID_ARG;
  if (B > LSS_BLOCK_MAX_ROWS || heads > 65536 || dim > 65536) return LSS_ERR_UNSUPPORTED;
  if (B == 0 || T == 0) return LSS_OK;
  if (!k || !v || !k_cache || !v_cache || !k_scale || !v_scale || !starts || !granted || !lens)
    return LSS_ERR_INVALID_ARG;
  if (!aligned_to(k_cache, 16) || !aligned_to(v_cache, 16)) return LSS_ERR_INVALID_ARG;
  AppendArgs a{k, v, k_token_stride, k_head_stride, v_token_stride, v_head_stride, k_cache, v_cache, k_scale,
               v_scale, num_blocks, heads, log2_of(block_size), dim, table, table_stride, width, starts, granted, lens, B, T, 0};
  const int per16 = dtype == LSS_DTYPE_F32 ? 4 : 8;  // values in 16 bytes
  a.aligned = aligned_to(k, 16) && aligned_to(v, 16) && k_token_stride % per16 == 0 && k_head_stride % per16 == 0 &&
              v_token_stride % per16 == 0 && v_head_stride % per16 == 0;
  // Blocks that a step can write: one per token at most, and two more per row than its tokens fill.
  const int64_t blocks = std::min((int64_t)T, (int64_t)T / block_size + 2 * (int64_t)B);
  const int64_t items = blocks * 2 * heads;
  const int dev = device_index(), smem = 4 * B;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  auto go = [&](auto kern, SmemSet& set, int team) {
    if (smem > 40 * 1024) {
      const cudaError_t e = allow_smem(kern, set, dev, smem);
      if (e != cudaSuccess) return e;
    }
    const int teams = KV_NT / 32 / team;
    const int64_t ctas = std::max((int64_t)1, std::min((items + teams - 1) / teams, (int64_t)sm_count(dev) * 3));
    return launch(kern, (unsigned)ctas, KV_NT, (size_t)smem, 1, false, st, a);
  };
  static SmemSet sets[9];
  // Warps per unit: as many as its values fill on the average (2048 a warp).
  const int64_t values = (int64_t)T * dim / blocks;
  const int team = values > 4096 ? 4 : values > 2048 + 512 ? 2 : 1;
  auto by_team = [&](auto k1, auto k2, auto k4, int at) {
    return status_of(team == 4 ? go(k4, sets[at + 2], 4) : team == 2 ? go(k2, sets[at + 1], 2) : go(k1, sets[at], 1));
  };
  switch (dtype) {
    case LSS_DTYPE_F32:
      return by_team(lss_append_kernel<LSS_DTYPE_F32, 1>, lss_append_kernel<LSS_DTYPE_F32, 2>, lss_append_kernel<LSS_DTYPE_F32, 4>, 0);
    case LSS_DTYPE_BF16:
      return by_team(lss_append_kernel<LSS_DTYPE_BF16, 1>, lss_append_kernel<LSS_DTYPE_BF16, 2>, lss_append_kernel<LSS_DTYPE_BF16, 4>, 3);
    default:
      return by_team(lss_append_kernel<LSS_DTYPE_F16, 1>, lss_append_kernel<LSS_DTYPE_F16, 2>, lss_append_kernel<LSS_DTYPE_F16, 4>, 6);
  }
}

size_t lss_attend_workspace_bytes(int dim) {
  switch (dim) {
    case 64: return std::max({attend_bytes<64, 1, 1>(), attend_bytes<64, 2, 1>(), attend_bytes<64, 4, 1>(), attend_tc_bytes<64>()});
    case 128: return std::max({attend_bytes<128, 1, 1>(), attend_bytes<128, 1, 2>(), attend_bytes<128, 2, 1>(), attend_bytes<128, 4, 1>(), attend_tc_bytes<128>()});
    case 256: return std::max(attend_bytes<256, 1, 1>(), attend_bytes<256, 2, 1>());
    default: return 0;
  }
}

int lss_attend(const void* q, int64_t q_token_stride, int64_t q_head_stride, int dtype, int T, int q_heads,
               int heads, int dim, const uint8_t* k_cache, const uint8_t* v_cache, const float* k_scale,
               const float* v_scale, int num_blocks, int block_size, const int32_t* table, int64_t table_stride,
               int width, const int32_t* starts, const int32_t* granted, const int32_t* lens, int B, float scale,
               void* out, int64_t out_token_stride, int64_t out_head_stride, float* lse, void* workspace,
               size_t workspace_bytes, void* stream) {
  return attend_entry<false>(q, q_token_stride, q_head_stride, dtype, T, q_heads, heads, dim, k_cache, v_cache, k_scale, v_scale, num_blocks, block_size, table, table_stride, width, starts, granted, lens, B, scale, out, out_token_stride, out_head_stride, lse, workspace, workspace_bytes, nullptr, stream);
}

}  // extern "C"
