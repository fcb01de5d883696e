// lss_attend_host.cuh — launches of the attention kernels: which one a row of the batch goes to.
#pragma once

#include "lss_attend_tc.cuh"
#include "lss_host.cuh"

static constexpr int AT_CAP_CTAS = 160;  // CTAs that the workspace has room for

template <int D, int NQ, int TP>
static inline size_t attend_bytes() {
  const size_t workers = (size_t)AT_CAP_CTAS * AtCfg<D, NQ, TP>::NW;
  return workers * (sizeof(int4) + 2 * at_piece(D, NQ) * sizeof(float));
}

template <int D, int DT, int NQ, int TP, bool TREE>
static inline cudaError_t launch_attend(AttendArgs a, void* ws, cudaStream_t st) {
  static SmemSet set;
  const int dev = device_index();
  constexpr int NW = AtCfg<D, NQ, TP>::NW;
  constexpr int smem = NW * AtCfg<D, NQ, TP>::ST * (32 * D + 16);
  cudaError_t e = allow_smem(lss_attend_kernel<D, DT, NQ, TP, TREE>, set, dev, smem);
  if (e != cudaSuccess) return e;
  // No more warps than there can be units.
  const int64_t groups = a.B + (int64_t)a.T * a.per / (8 * NQ) + 1;
  const int64_t units = groups * a.heads * ((((int64_t)a.width << a.bs_shift) + 15) >> 4);
  const int ctas = (int)std::min((int64_t)std::min(sm_count(dev), AT_CAP_CTAS), (units + NW - 1) / NW);
  a.meta = reinterpret_cast<int4*>(ws);
  a.part = reinterpret_cast<float*>(a.meta + (size_t)ctas * NW);
  // Two tiles a warp and less on eight SMs: one launch (a call for one short request 20.6 -> 17.5 us on the host); with
  // more tiles eight SMs' share of the bandwidth would cost more than the second launch.
  a.fused = units <= 8 * NW * 2;
  if (a.fused) {
    const int size = ctas <= 1 ? 1 : ctas <= 2 ? 2 : ctas <= 4 ? 4 : 8;
    return launch(lss_attend_kernel<D, DT, NQ, TP, TREE>, (unsigned)size, NW * 32, smem, size, false, st, a);
  }
  e = launch(lss_attend_kernel<D, DT, NQ, TP, TREE>, (unsigned)ctas, NW * 32, smem, 1, false, st, a);
  if (e != cudaSuccess) return e;
  return launch(lss_attend_join_kernel<D, DT, NQ, TP, TREE>, (unsigned)(ctas * NW), 256, 0, 1, true, st, a);
}

template <int D>
static inline size_t attend_tc_bytes() {
  return (size_t)AT_CAP_CTAS * (sizeof(int4) + 2 * pa_piece(D) * sizeof(float));
}

template <int D, int DT, bool TREE>
static inline cudaError_t launch_attend_tc(AttendArgs a, void* ws, cudaStream_t st) {
  static SmemSet set;
  const int dev = device_index();
  constexpr int smem = pa_smem(D);
  cudaError_t e = allow_smem(lss_attend_tc_kernel<D, DT, TREE>, set, dev, smem);
  if (e != cudaSuccess) return e;
  const int ctas = std::min(sm_count(dev), AT_CAP_CTAS);
  a.meta = reinterpret_cast<int4*>(ws);
  a.part = reinterpret_cast<float*>(a.meta + AT_CAP_CTAS);
  e = launch(lss_attend_tc_kernel<D, DT, TREE>, (unsigned)ctas, PA_NT, smem, 1, false, st, a);
  if (e != cudaSuccess) return e;
  return launch(lss_attend_tc_join_kernel<D, DT, TREE>, (unsigned)(ctas * (PA_ROWS / 32)), 256, 0, 1, true, st, a);
}

// `rows`: query rows per key head that a row of the batch has.
template <int D, int DT, bool TREE>
static inline cudaError_t launch_attend_few(const AttendArgs& a, int64_t rows, void* ws, cudaStream_t st) {
  if (rows <= 8) {
    // Long contexts take two tiles a step (AtCfg); how long they are only the table's width tells here.
    if constexpr (D == 128) {
      if (((int64_t)a.width << a.bs_shift) >= 1024) return launch_attend<D, DT, 1, 2, TREE>(a, ws, st);
    }
    return launch_attend<D, DT, 1, 1, TREE>(a, ws, st);
  }
  if constexpr (TREE) {
    // Small trees: groups of eight rows where all of their tiles find a warp at once (6 tokens of 7 heads per key head of 64
    // over 700: 15 us, in groups of 16 20 us, of 32 26 us).
    const int64_t units = (a.B + (int64_t)a.T * a.per / 8 + 1) * a.heads * ((((int64_t)a.width << a.bs_shift) + 15) >> 4);
    if (units <= (int64_t)sm_count(device_index()) * AtCfg<D, 1, 1>::NW) return launch_attend<D, DT, 1, 1, TREE>(a, ws, st);
  }
  if constexpr (D < 256) {
    if (rows > 16) return launch_attend<D, DT, 4, 1, TREE>(a, ws, st);
  }
  return launch_attend<D, DT, 2, 1, TREE>(a, ws, st);
}

// A step of single tokens has `per` query rows per key head and row; else the average decides.  A step with more
// tokens than rows, and enough of them to fill the SMs, may mix prompt chunks, rows of a few tokens and single
// tokens, and only the device knows which is which: rows of enough query rows go to the tensor-memory kernel, the others to the
// one for few rows, one launch after the other on the same workspace.  Its group is that of a single token, or of 16 rows where the average
// row is a short one (trees: always).  In tensor memory a row costs about the same up to 128 query rows, but more for its start and end; for few
// rows it costs once more for every 16.  Measured with 8 key heads of 4 queries, us in tensor memory (in groups of 16):
//   D = 128, 17 to 32 query rows: 64 rows over 1,000 tokens 115 (109-115), 2,000 170 (164-170), 4,000 243 (268-274); 512 over 300 455 (264)
//   33 to 48: 64 rows over 1,000 121 (133), 2,000 178 (219), 4,000 250 (375); 512 over 100 344 (156), 300 436 (373), 600 516-547 (524-537)
//   D = 64, 33 to 48: 64 rows over 1,000 94 (94), 2,000 143 (131), 4,000 203 (211); 512 over 300 356 (209)
//   49 to 63: 64 rows over 2,000 147 (166), 4,000 215 (270); 512 over 300 379 (270), 1,000 520-553 (563)
//   rows over 50 to 16,000, D = 128, all by these borders: 5, 8, 9, 12, 16 tokens 477, 483, 491, 481, 463
// so that lengths from AT_LONG and at_long_more on decide below rows_any.  Causal steps of more than 8 heads per key head have one border, above a
// single token's rows.  Single tokens beside one chunk of 449 pay for the second launch (10 us).
// A step of no more tokens than rows counts as one of single tokens: a chunk among idle rows is right, but goes in
// their groups (200 tokens over 8,000 beside 255 idle rows 213 us, alone 201; 500 beside 511 507 us, alone 171), as the
// launches for chunks would cost every step of single tokens 8 to 10 us.
// Trees: the rows of a batch are mostly alike, a few tokens to some dozens each, so that a single row may have tokens enough for the SMs too
// (64 tokens of 8 heads per key head over 20,000 alone 119 us, 300 in groups of 16), and in a batch of large ones the small ones
// go along (48 of 8 to 32 tokens over 50 to 8,000: 206 us, in the same run 222 with a second launch for a few rows).
template <int D, int DT, bool TREE>
static inline cudaError_t launch_attend_rows(AttendArgs a, void* ws, cudaStream_t st) {
  const int64_t average = (int64_t)a.per * ((a.T + (int64_t)a.B - 1) / a.B);
  a.side = 0;
  if constexpr (D < 256) {
    const int sms = sm_count(device_index());
    const bool low = TREE || a.per <= 8;
    a.rows_any = low && D == 128 ? 49 : 64;
    a.long_more = at_long_more(D);
    a.rows_long = low ? (D == 128 ? 17 : 33) : 64;
    if (TREE && average >= a.rows_any) a.rows_any = a.rows_long;
    const int usual = ((int64_t)a.width << a.bs_shift) >= AT_LONG ? a.rows_long : a.rows_any;
    const int64_t tiles = ((((int64_t)a.width << a.bs_shift) + PA_KT - 1) / PA_KT) * a.heads * a.B;
    if (a.T > a.B && ((int64_t)a.heads * a.per * a.T >= (int64_t)PA_ROWS * sms / 4 || (TREE && average >= usual && tiles >= sms))) {
      a.side = 1;
      const cudaError_t e = launch_attend_tc<D, DT, TREE>(a, ws, st);
      if (e != cudaSuccess) return e;
      a.side = 2;
      return launch_attend_few<D, DT, TREE>(a, TREE || average < 64 ? std::max((int64_t)a.per, std::min(average, (int64_t)16)) : a.per, ws, st);
    }
  }
  return launch_attend_few<D, DT, TREE>(a, average, ws, st);
}

template <int D, bool TREE>
static inline cudaError_t launch_attend_dt(int dtype, const AttendArgs& a, void* ws, cudaStream_t st) {
  return dtype == LSS_DTYPE_BF16 ? launch_attend_rows<D, LSS_DTYPE_BF16, TREE>(a, ws, st) : launch_attend_rows<D, LSS_DTYPE_F16, TREE>(a, ws, st);
}

// Checks and launch of lss_attend and lss_attend_tree.
template <bool TREE>
static inline int attend_entry(const void* q, int64_t q_token_stride, int64_t q_head_stride, int dtype, int T, int q_heads,
               int heads, int dim, const uint8_t* k_cache, const uint8_t* v_cache, const float* k_scale,
               const float* v_scale, int num_blocks, int block_size, const int32_t* table, int64_t table_stride,
               int width, const int32_t* starts, const int32_t* granted, const int32_t* lens, int B, float scale,
               void* out, int64_t out_token_stride, int64_t out_head_stride, float* lse, void* workspace,
               size_t workspace_bytes, const int32_t* span, void* stream) {
  if ((dtype != LSS_DTYPE_BF16 && dtype != LSS_DTYPE_F16) || T < 0 || heads < 1 || q_heads < heads ||
      q_heads % heads != 0 || !block_size_ok(block_size))
    return LSS_ERR_INVALID_ARG;
  if (q_token_stride < 0 || q_head_stride < 0 || out_token_stride < 0 || out_head_stride < dim) return LSS_ERR_INVALID_ARG;
  if (!table_ok(table, table_stride, width, B, block_size, num_blocks)) return LSS_ERR_INVALID_ARG;
  if (dim != 64 && dim != 128 && dim != 256) return LSS_ERR_UNSUPPORTED;
  if (heads > 65536 || (int64_t)T * q_heads > (1 << 30)) return LSS_ERR_UNSUPPORTED;
  if (B == 0 || T == 0) return LSS_OK;
  if (TREE && (!span || !aligned_to(span, 8))) return LSS_ERR_INVALID_ARG;
  if (!q || !out || !k_cache || !v_cache || !k_scale || !v_scale || !starts || !granted || !lens)
    return LSS_ERR_INVALID_ARG;
  if (!aligned_to(k_cache, 16) || !aligned_to(v_cache, 16)) return LSS_ERR_INVALID_ARG;
  if (T > 1 && out_token_stride < (q_heads - 1) * out_head_stride + dim &&
      (out_token_stride < dim || out_head_stride < (T - 1) * out_token_stride + dim))
    return LSS_ERR_INVALID_ARG;  // rows of the result lie over each other, whether tokens or heads are outside
  if (rows_shifted(q, 2 * q_token_stride, 2 * q_head_stride, out, 2 * out_token_stride, 2 * out_head_stride, T, q_heads, 2 * (int64_t)dim))
    return LSS_ERR_INVALID_ARG;
  if (!workspace || workspace_bytes < lss_attend_workspace_bytes(dim) || !aligned_to(workspace, 16)) return LSS_ERR_WORKSPACE;
  AttendArgs a{};
  a.q = q;
  a.q_st = q_token_stride;
  a.q_sh = q_head_stride;
  a.out = out;
  a.o_st = out_token_stride;
  a.o_sh = out_head_stride;
  a.lse = lse;
  a.kc = k_cache;
  a.vc = v_cache;
  a.ks = k_scale;
  a.vs = v_scale;
  a.num_blocks = num_blocks;
  a.heads = heads;
  a.per = q_heads / heads;
  a.bs_shift = log2_of(block_size);
  a.table = table;
  a.table_stride = table_stride;
  a.width = width;
  a.starts = starts;
  a.granted = granted;
  a.lens = lens;
  a.B = B;
  a.T = T;
  a.scale = scale * LOG2E;
  a.span = reinterpret_cast<const int2*>(span);
  a.aligned = aligned_to(q, 16) && aligned_to(out, 16) && q_token_stride % 8 == 0 && q_head_stride % 8 == 0 &&
              out_token_stride % 8 == 0 && out_head_stride % 8 == 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  switch (dim) {
    case 64: return status_of(launch_attend_dt<64, TREE>(dtype, a, workspace, st));
    case 128: return status_of(launch_attend_dt<128, TREE>(dtype, a, workspace, st));
    default: return status_of(launch_attend_dt<256, TREE>(dtype, a, workspace, st));
  }
}
