// lss_drafts.cu — C ABI of the decode-step operators around drafted tokens and shared blocks: norms
// with the position rotation, trees and their acceptance, tokens and blocks moved, shared and returned.
#include "lss_host.cuh"
#include "lss_kvmove.cuh"
#include "lss_rotate.cuh"
#include "lss_share.cuh"
#include "lss_tree.cuh"

// Two arrays of T tokens (start, bytes between tokens, between heads, heads) of which some head lies over one of the
// other's.  With equal strides exactly, so that heads of the two may take turns; else by the extents of their tokens' heads.
static bool tokens_overlap(const void* x, int64_t x_st, int64_t x_sh, int x_heads, const void* y, int64_t y_st, int64_t y_sh, int y_heads,
                           int T, int64_t n) {
  if (!rows_overlap(x, x_st, (x_heads - 1) * x_sh + n, y, y_st, (y_heads - 1) * y_sh + n, T)) return false;
  if (T == 1) x_st = y_st = 0;  // one token, one head: the stride says nothing
  if (x_heads == 1) x_sh = y_sh;
  if (y_heads == 1) y_sh = x_sh;
  if (x_st != y_st || x_sh != y_sh) return true;
  return rows_meet((int64_t)(reinterpret_cast<intptr_t>(y) - reinterpret_cast<intptr_t>(x)), x_st, x_sh, T, T, x_heads, y_heads, n);
}

template <int DT, int N, int L, bool PAIRS>
static cudaError_t launch_rotate(const RotateArgs& a, cudaStream_t st) {
  const int teams = RO_NT / L, sms = sm_count(device_index());
  // Tokens per CTA, a power of two.  A wave of three CTAs per SM takes about as long as its teams' heads and four more
  // (start, weights, sines): 1,000 tokens of 32 + 8 heads of 128 one by one 22 us, four by four 14; 8,192 by 8 or 32 39 us, by 16 45 (alone, cold caches).
  int tk = 1;
  int64_t best = INT64_MAX;
  for (int t = 1; t <= teams; t *= 2) {
    const int per = teams / t, ctas = (a.T + t - 1) / t;
    const int64_t cost = (int64_t)((ctas + 3 * sms - 1) / (3 * sms)) * (4 + (a.side[0].heads + per - 1) / per + (a.side[1].heads + per - 1) / per);
    if (cost < best) {
      best = cost;
      tk = t;
    }
  }
  const int ring = N > 1 ? RO_ST * 2 * 16 * RO_NT : 0;
  const int smem = ring + a.dim * 8 + tk * a.half * 8;
  static SmemSet set;
  const cudaError_t e = allow_smem(lss_rotate_kernel<DT, N, L, PAIRS>, set, device_index(), smem);
  if (e != cudaSuccess) return e;
  return launch(lss_rotate_kernel<DT, N, L, PAIRS>, (unsigned)((a.T + tk - 1) / tk), RO_NT, smem, 1, false, st, a, tk);
}
template <int DT, bool PAIRS>
static cudaError_t launch_rotate_dim(const RotateArgs& a, bool wide, cudaStream_t st) {
  constexpr int N = DT == LSS_DTYPE_F32 ? 4 : 8;  // values in 16 bytes
  if (!wide) return launch_rotate<DT, 1, 32, PAIRS>(a, st);
  if (a.dim <= 8 * N) return launch_rotate<DT, N, 4, PAIRS>(a, st);
  if (a.dim <= 16 * N) return launch_rotate<DT, N, 8, PAIRS>(a, st);
  if (a.dim <= 32 * N) return launch_rotate<DT, N, 16, PAIRS>(a, st);
  return launch_rotate<DT, N, 32, PAIRS>(a, st);
}
template <int DT>
static cudaError_t launch_rotate_dt(const RotateArgs& a, bool wide, cudaStream_t st) {
  return a.interleaved ? launch_rotate_dim<DT, true>(a, wide, st) : launch_rotate_dim<DT, false>(a, wide, st);
}

static bool rows_ok(const void* x, int64_t st, int64_t sh, int heads, int T, int dim) {
  // rows of a result lie over each other, whether tokens or heads are outside
  return x && st >= 0 && sh >= 0 && (heads == 1 || sh >= dim) && (T == 1 || st >= dim) &&
         (T == 1 || heads == 1 || st >= (heads - 1) * sh + dim || sh >= (T - 1) * st + dim);
}

// CTAs that share a release: every entry is a scattered access or two per pass, which eight SMs take longer for than
// sixteen (37 us against 23 for 46,000 entries); sixteen where the device runs such a cluster with all of its shared memory.
static int give_ctas(int dev) {
  static int n[MAX_DEV] = {};
  std::lock_guard<std::mutex> lock(g_mu);
  if (n[dev] == 0) {
    constexpr int smem = 224 * 1024;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(16, 1, 1);
    cfg.blockDim = dim3(BL_NT, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 16;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    int c = 0;
    const bool ok = cudaFuncSetAttribute(lss_give_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess &&
                    cudaFuncSetAttribute(lss_give_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) == cudaSuccess &&
                    cudaOccupancyMaxActiveClusters(&c, lss_give_kernel, &cfg) == cudaSuccess && c >= 1;
    if (!ok) cudaGetLastError();
    n[dev] = ok ? 16 : BL_MAXCL;
  }
  return n[dev];
}

extern "C" {

int lss_norm_rotate(const void* q, int64_t q_token_stride, int64_t q_head_stride, void* q_out, int64_t q_out_token_stride,
                    int64_t q_out_head_stride, int q_heads, const void* k, int64_t k_token_stride, int64_t k_head_stride,
                    void* k_out, int64_t k_out_token_stride, int64_t k_out_head_stride, int k_heads, int dtype, int T, int dim,
                    const int32_t* positions, const float* freqs, int rot, int interleaved, const void* q_weight,
                    const void* k_weight, int weight_dtype, float eps, void* stream) {
  if (!known_dtype(dtype) || T < 0 || q_heads < 1 || k_heads < 1 || dim < 2 || dim % 2 != 0 || rot < 0 || rot % 2 != 0 || rot > dim)
    return LSS_ERR_INVALID_ARG;
  if ((q_weight || k_weight) && !known_dtype(weight_dtype)) return LSS_ERR_INVALID_ARG;
  if (q_token_stride < 0 || q_head_stride < 0 || k_token_stride < 0 || k_head_stride < 0) return LSS_ERR_INVALID_ARG;
  if (dim > 512 || q_heads > 65536 || k_heads > 65536 || (int64_t)T * (q_heads + k_heads) > (1 << 30)) return LSS_ERR_UNSUPPORTED;
  if (T == 0) return LSS_OK;
  if (!q || !k || !positions || (rot > 0 && !freqs)) return LSS_ERR_INVALID_ARG;
  if (!rows_ok(q_out, q_out_token_stride, q_out_head_stride, q_heads, T, dim) ||
      !rows_ok(k_out, k_out_token_stride, k_out_head_stride, k_heads, T, dim))
    return LSS_ERR_INVALID_ARG;
  const int64_t e = dtype == LSS_DTYPE_F32 ? 4 : 2, n = dim * e;
  if (rows_shifted(q, q_token_stride * e, q_head_stride * e, q_out, q_out_token_stride * e, q_out_head_stride * e, T, q_heads, n) ||
      rows_shifted(k, k_token_stride * e, k_head_stride * e, k_out, k_out_token_stride * e, k_out_head_stride * e, T, k_heads, n) ||
      tokens_overlap(q, q_token_stride * e, q_head_stride * e, q_heads, k_out, k_out_token_stride * e, k_out_head_stride * e, k_heads, T, n) ||
      tokens_overlap(k, k_token_stride * e, k_head_stride * e, k_heads, q_out, q_out_token_stride * e, q_out_head_stride * e, q_heads, T, n) ||
      tokens_overlap(q_out, q_out_token_stride * e, q_out_head_stride * e, q_heads, k_out, k_out_token_stride * e, k_out_head_stride * e,
                     k_heads, T, n))
    return LSS_ERR_INVALID_ARG;
  RotateArgs a{};
  a.side[0] = {q, q_out, q_weight, q_token_stride, q_head_stride, q_out_token_stride, q_out_head_stride, q_heads};
  a.side[1] = {k, k_out, k_weight, k_token_stride, k_head_stride, k_out_token_stride, k_out_head_stride, k_heads};
  a.positions = positions;
  a.freqs = freqs;
  a.T = T;
  a.dim = dim;
  a.half = rot / 2;
  a.w_dtype = weight_dtype;
  a.interleaved = interleaved != 0;
  a.eps = eps;
  // 16 bytes at a time where all groups of values lie on 16-byte boundaries and turn with one other group; f32 up to
  // a dim of 256 (a lane's 8 values times 32).
  bool wide = dim % 16 == 0 && a.half % 8 == 0 && dim * e <= 1024;
  for (const RotateSide& s : a.side) {
    const int64_t per16 = 16 / e;
    wide = wide && aligned_to(s.x, 16) && aligned_to(s.y, 16) && s.x_st % per16 == 0 && s.x_sh % per16 == 0 && s.y_st % per16 == 0 &&
           s.y_sh % per16 == 0;
  }
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  switch (dtype) {
    case LSS_DTYPE_F32: return status_of(launch_rotate_dt<LSS_DTYPE_F32>(a, wide, st));
    case LSS_DTYPE_BF16: return status_of(launch_rotate_dt<LSS_DTYPE_BF16>(a, wide, st));
    default: return status_of(launch_rotate_dt<LSS_DTYPE_F16>(a, wide, st));
  }
}

int lss_tree_plan(const int32_t* starts, const int32_t* granted, const int32_t* lens, int B, const int32_t* parents, int T,
                  int32_t* span, int32_t* positions, void* stream) {
  if (B < 0 || T < 0) return LSS_ERR_INVALID_ARG;
  if (B > LSS_BLOCK_MAX_ROWS) return LSS_ERR_UNSUPPORTED;
  if (T == 0) return LSS_OK;
  if (!parents || !span || !aligned_to(span, 8) || !positions || (B > 0 && (!starts || !granted || !lens))) return LSS_ERR_INVALID_ARG;
  TreeArgs a{starts, granted, lens, parents, reinterpret_cast<int2*>(span), positions, B, T};
  return status_of(launch(lss_tree_kernel, (unsigned)B + 1, TR_NT, 0, 1, false, reinterpret_cast<cudaStream_t>(stream), a));
}

int lss_tree_accept(const int32_t* starts, const int32_t* granted, const int32_t* lens, int B, const int32_t* parents,
                    const int32_t* drafts, const int32_t* targets, const int32_t* codes, const int32_t* given, int T, int32_t* path,
                    int32_t* tokens, int32_t* counts, int32_t* lens_out, int32_t* last, int32_t* codes_out, void* stream) {
  if (B < 0 || T < 0) return LSS_ERR_INVALID_ARG;
  if (B > LSS_BLOCK_MAX_ROWS) return LSS_ERR_UNSUPPORTED;
  if (T > 0 && (!parents || !drafts || !targets || !path || !tokens)) return LSS_ERR_INVALID_ARG;
  if (B > 0 && (!starts || !granted || !lens || !counts || !lens_out || !last || !codes_out)) return LSS_ERR_INVALID_ARG;
  if (B > 0 && (cut(lens_out, lens, B) || lens_out == granted || cut(lens_out, granted, B))) return LSS_ERR_INVALID_ARG;
  if (B == 0 && T == 0) return LSS_OK;
  AcceptArgs a{starts, granted, lens, parents, drafts, targets, codes, given, path, tokens, counts, lens_out, last, codes_out, B, T};
  return status_of(launch(lss_accept_kernel, (unsigned)(B / (AC_NT / 32) + 1), AC_NT, 0, 1, false, reinterpret_cast<cudaStream_t>(stream), a));
}

int lss_kv_compact(uint8_t* k_cache, uint8_t* v_cache, float* k_scale, float* v_scale, int num_blocks, int heads, int block_size,
                   int dim, const int32_t* table, int64_t table_stride, int width, const int32_t* starts, const int32_t* granted,
                   const int32_t* lens, int B, const int32_t* path, const int32_t* counts, int T, void* stream) {
  if (T < 0 || heads < 1 || dim < 8 || dim % 8 != 0 || !block_size_ok(block_size)) return LSS_ERR_INVALID_ARG;
  if (!table_ok(table, table_stride, width, B, block_size, num_blocks)) return LSS_ERR_INVALID_ARG;
  if (B > LSS_BLOCK_MAX_ROWS || heads > 65536 || dim > 65536) return LSS_ERR_UNSUPPORTED;
  if (B == 0 || T == 0) return LSS_OK;
  if (!k_cache || !v_cache || !k_scale || !v_scale || !starts || !granted || !lens || !path || !counts) return LSS_ERR_INVALID_ARG;
  if (!aligned_to(k_cache, 16) || !aligned_to(v_cache, 16)) return LSS_ERR_INVALID_ARG;
  CompactArgs a{k_cache, v_cache, k_scale, v_scale, num_blocks, heads, log2_of(block_size), dim, table, table_stride, width, starts,
                granted, lens, path, counts, B, T};
  const int64_t ctas = ((int64_t)B * 2 * heads + MV_NT / 32 - 1) / (MV_NT / 32);
  if (ctas > INT32_MAX) return LSS_ERR_UNSUPPORTED;
  return status_of(launch(lss_compact_kernel, (unsigned)ctas, MV_NT, 0, 1, false, reinterpret_cast<cudaStream_t>(stream), a));
}

int lss_kv_copy(uint8_t* k_cache, uint8_t* v_cache, float* k_scale, float* v_scale, int num_blocks, int heads, int block_size,
                int dim, const int32_t* copies, int n, void* stream) {
  if (n < 0 || num_blocks < 1 || heads < 1 || dim < 8 || dim % 8 != 0 || !block_size_ok(block_size)) return LSS_ERR_INVALID_ARG;
  if (heads > 65536 || dim > 65536) return LSS_ERR_UNSUPPORTED;
  if (n == 0) return LSS_OK;
  if (!k_cache || !v_cache || !k_scale || !v_scale || !copies) return LSS_ERR_INVALID_ARG;
  if (!aligned_to(k_cache, 16) || !aligned_to(v_cache, 16)) return LSS_ERR_INVALID_ARG;
  const int64_t pieces = (int64_t)heads * block_size * dim / 16, parts = (pieces + CP_NT * CP_PER - 1) / (CP_NT * CP_PER);
  if (parts * 2 * n > INT32_MAX) return LSS_ERR_UNSUPPORTED;
  CopyArgs a{k_cache, v_cache, k_scale, v_scale, num_blocks, heads, pieces, copies, n, (int)parts};
  return status_of(launch(lss_copy_kernel, (unsigned)(parts * 2 * n), CP_NT, 0, 1, false, reinterpret_cast<cudaStream_t>(stream), a));
}

int lss_block_fork(int32_t* table, int64_t table_stride, int width, const int32_t* lens, int B, int block_size,
                   const int32_t* src_rows, const int32_t* dst_rows, const int32_t* upto, int n, int32_t* shares,
                   const int32_t* free_blocks, int num_blocks, const int32_t* n_free, int32_t* granted, int32_t* copies,
                   int32_t* lens_out, int32_t* n_free_out, void* stream) {
  if (!table_ok(table, table_stride, width, B, block_size, num_blocks) || n < 0) return LSS_ERR_INVALID_ARG;
  if (B > LSS_BLOCK_MAX_ROWS || n > LSS_BLOCK_MAX_ROWS) return LSS_ERR_UNSUPPORTED;
  if (!shares || !free_blocks || !n_free || !n_free_out || (B > 0 && (!lens || !lens_out))) return LSS_ERR_INVALID_ARG;
  if (n > 0 && (!src_rows || !dst_rows || !granted || !copies)) return LSS_ERR_INVALID_ARG;
  if (cut(lens_out, lens, B)) return LSS_ERR_INVALID_ARG;
  ForkArgs a{table, table_stride, width, lens, src_rows, dst_rows, upto, n, B, block_size, num_blocks, shares, free_blocks, n_free,
             granted, copies, lens_out, n_free_out};
  static SmemSet set;
  const int smem = 4 * B;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (smem > 40 * 1024) {
    const cudaError_t e = allow_smem(lss_fork_kernel, set, device_index(), smem);
    if (e != cudaSuccess) return status_of(e);
  }
  cudaError_t e = launch(lss_fork_kernel, 1, BL_NT, (size_t)smem, 1, false, st, a);
  if (e == cudaSuccess && n > 0) e = launch(lss_fork_table_kernel, (unsigned)n, FK_NT, 0, 1, true, st, a);
  return status_of(e);
}

int lss_block_give(const int32_t* table, int64_t table_stride, int width, const int32_t* lens, const int32_t* codes,
                   const int32_t* keep, int B, int block_size, int32_t* shares, int32_t* free_blocks, int num_blocks,
                   const int32_t* n_free, int32_t* lens_out, int32_t* n_free_out, void* stream) {
  if (!table_ok(table, table_stride, width, B, block_size, num_blocks)) return LSS_ERR_INVALID_ARG;
  if (B > LSS_BLOCK_MAX_ROWS || (int64_t)B * width > (1 << 30)) return LSS_ERR_UNSUPPORTED;
  if (!free_blocks || !n_free || !n_free_out || (B > 0 && (!lens || !lens_out))) return LSS_ERR_INVALID_ARG;
  if (cut(lens_out, lens, B) || (codes && cut(lens_out, codes, B)) || (keep && cut(lens_out, keep, B))) return LSS_ERR_INVALID_ARG;
  GiveArgs a{table, table_stride, width, lens, codes, keep, B, block_size, num_blocks, shares, free_blocks, n_free, lens_out, n_free_out, 0};
  static SmemSet set;
  const int dev = device_index(), ctas = cluster_for((B + 31) / 32, give_ctas(dev));
  // Room for the entries of each warp's rows, up to 192 KB per CTA.
  const int64_t pieces = (int64_t)((B + ctas * 32 - 1) / (ctas * 32)) * (((int64_t)width + 255) / 256);
  a.held = (int)std::min(pieces, (int64_t)(224 * 1024 - 4 * B) / (32 * 1024));
  const int smem = 4 * B + a.held * 32 * 1024;
  if (smem > 40 * 1024) {
    const cudaError_t e = allow_smem(lss_give_kernel, set, dev, smem);
    if (e != cudaSuccess) return status_of(e);
  }
  return status_of(launch(lss_give_kernel, (unsigned)ctas, BL_NT, (size_t)smem, ctas, false, reinterpret_cast<cudaStream_t>(stream), a));
}

}  // extern "C"
