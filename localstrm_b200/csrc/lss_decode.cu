// lss_decode.cu — C ABI of the decode-step operators around the sampler: 4-bit products, block
// tables, the 8-bit key/value cache and its attention.
#include <algorithm>
#include <cstdlib>
#include <mutex>
#include <utility>

#include "lss_attend_tc.cuh"
#include "lss_blocks.cuh"
#include "lss_int4_tc.cuh"
#include "lss_kvcache.cuh"

using namespace lss;

static constexpr int MAX_DEV = 64;

static int device_index() {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= MAX_DEV) dev = 0;
  return dev;
}

static std::mutex g_mu;

static int sm_count(int dev) {
  static int n[MAX_DEV] = {};
  std::lock_guard<std::mutex> lock(g_mu);
  if (n[dev] == 0 && (cudaDeviceGetAttribute(&n[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n[dev] < 1)) {
    cudaGetLastError();
    n[dev] = 0;
    return 148;
  }
  return n[dev];
}

// Raises a kernel's dynamic shared memory limit, once per device and size.
struct SmemSet {
  int bytes[MAX_DEV] = {};
};
template <class K>
static cudaError_t allow_smem(K kern, SmemSet& set, int dev, int bytes) {
  std::lock_guard<std::mutex> lock(g_mu);
  if (bytes <= set.bytes[dev]) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) set.bytes[dev] = bytes;
  return e;
}

template <class... KA, class... A>
static cudaError_t launch(void (*kern)(KA...), unsigned grid, unsigned block, size_t smem, int cluster, bool pdl,
                          cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid, 1, 1);
  cfg.blockDim = dim3(block, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  int na = 0;
  if (cluster > 1) {
    at[na].id = cudaLaunchAttributeClusterDimension;
    at[na].val.clusterDim.x = (unsigned)cluster;
    at[na].val.clusterDim.y = 1;
    at[na].val.clusterDim.z = 1;
    ++na;
  }
  if (pdl) {
    at[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[na].val.programmaticStreamSerializationAllowed = 1;
    ++na;
  }
  cfg.attrs = at;
  cfg.numAttrs = (unsigned)na;
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

static int status_of(cudaError_t e) {
  if (e == cudaSuccess) return LSS_OK;
  cudaGetLastError();
  return LSS_ERR_CUDA;
}

static bool aligned_to(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
static bool known_dtype(int d) { return d == LSS_DTYPE_F32 || d == LSS_DTYPE_BF16 || d == LSS_DTYPE_F16; }
static bool block_size_ok(int bs) { return bs == 16 || bs == 32 || bs == 64 || bs == 128 || bs == 256; }
// Rows of two matrices (start, bytes between rows, bytes of a row) that share memory.  Rows of one pitch may lie
// beside each other.
static bool rows_overlap(const void* x, int64_t x_pitch, int64_t x_row, const void* y, int64_t y_pitch, int64_t y_row, int rows) {
  const int64_t d = (int64_t)(reinterpret_cast<intptr_t>(y) - reinterpret_cast<intptr_t>(x));
  if (d >= (rows - 1) * x_pitch + x_row || -d >= (rows - 1) * y_pitch + y_row) return false;
  if (rows == 1 || x_pitch != y_pitch) return true;
  const int64_t at = (d % x_pitch + x_pitch) % x_pitch;  // where y's rows start in x's pitch
  return at < x_row || at + y_row > x_pitch;
}
// Two arrays of T x H rows of n bytes (start, bytes between tokens and between heads) that share memory without
// being the same rows: a result would be written where another CTA still reads its query.  With equal strides
// exactly, else wherever the extents meet.
static bool rows_shifted(const void* x, int64_t x_st, int64_t x_sh, const void* y, int64_t y_st, int64_t y_sh, int64_t T, int64_t H, int64_t n) {
  if (T == 1) x_st = y_st = 0;  // one token, one head: the stride says nothing
  if (H == 1) x_sh = y_sh = 0;
  const int64_t d = (int64_t)(reinterpret_cast<intptr_t>(y) - reinterpret_cast<intptr_t>(x));
  if (d >= (T - 1) * x_st + (H - 1) * x_sh + n || -d >= (T - 1) * y_st + (H - 1) * y_sh + n) return false;
  if (x_st != y_st || x_sh != y_sh) return true;
  if (d == 0) return false;
  if (T < H) {  // the walk below is over the shorter side
    std::swap(T, H);
    std::swap(x_st, x_sh);
  }
  for (int64_t j = 1 - H; j < H; ++j) {  // rows i tokens and j heads apart begin d - i st - j sh bytes apart
    const int64_t r = d - j * x_sh, i0 = x_st > 0 ? (r >= 0 ? r / x_st : -((-r + x_st - 1) / x_st)) : 0;
    for (int64_t i = i0; i <= i0 + 1; ++i)
      if (i > -T && i < T && std::abs(r - i * x_st) < n) return true;
  }
  return false;
}
// Arrays of n entries of which one begins inside the other.
static bool cut(const int32_t* x, const int32_t* y, int64_t n) { return x != y && x < y + n && y < x + n; }
static int log2_of(int v) {
  int s = 0;
  while ((1 << s) < v) ++s;
  return s;
}
static int cluster_for(int64_t ctas, int most) {
  int c = 1;
  while (c < most && c < ctas) c <<= 1;
  return c;
}

// ---------------------------------------------------------------- block tables
static bool table_ok(const void* table, int64_t stride, int width, int B, int bs, int num_blocks) {
  return (table || B == 0) && width >= 1 && stride >= width && B >= 0 && bs >= 1 && num_blocks >= 1 &&
         (int64_t)width * bs <= (1 << 30);
}

// ---------------------------------------------------------------- attention
static constexpr int AT_CAP_CTAS = 160;  // CTAs that the workspace has room for

template <int D, int NQ, int TP>
static size_t attend_bytes() {
  const size_t workers = (size_t)AT_CAP_CTAS * AtCfg<D, NQ, TP>::NW;
  return workers * (sizeof(int4) + 2 * at_piece(D, NQ) * sizeof(float));
}

template <int D, int DT, int NQ, int TP = 1>
static cudaError_t launch_attend(AttendArgs a, void* ws, cudaStream_t st) {
  static SmemSet set;
  const int dev = device_index();
  constexpr int NW = AtCfg<D, NQ, TP>::NW;
  constexpr int smem = NW * AtCfg<D, NQ, TP>::ST * (32 * D + 16);
  cudaError_t e = allow_smem(lss_attend_kernel<D, DT, NQ, TP>, set, dev, smem);
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
    return launch(lss_attend_kernel<D, DT, NQ, TP>, (unsigned)size, NW * 32, smem, size, false, st, a);
  }
  e = launch(lss_attend_kernel<D, DT, NQ, TP>, (unsigned)ctas, NW * 32, smem, 1, false, st, a);
  if (e != cudaSuccess) return e;
  return launch(lss_attend_join_kernel<D, DT, NQ, TP>, (unsigned)(ctas * NW), 256, 0, 1, true, st, a);
}

template <int D>
static size_t attend_tc_bytes() {
  return (size_t)AT_CAP_CTAS * (sizeof(int4) + 2 * pa_piece(D) * sizeof(float));
}

template <int D, int DT>
static cudaError_t launch_attend_tc(AttendArgs a, void* ws, cudaStream_t st) {
  static SmemSet set;
  const int dev = device_index();
  constexpr int smem = 1024 + 6 * 128 * D * 2;
  cudaError_t e = allow_smem(lss_attend_tc_kernel<D, DT>, set, dev, smem);
  if (e != cudaSuccess) return e;
  const int ctas = std::min(sm_count(dev), AT_CAP_CTAS);
  a.meta = reinterpret_cast<int4*>(ws);
  a.part = reinterpret_cast<float*>(a.meta + AT_CAP_CTAS);
  e = launch(lss_attend_tc_kernel<D, DT>, (unsigned)ctas, PA_NT, smem, 1, false, st, a);
  if (e != cudaSuccess) return e;
  return launch(lss_attend_tc_join_kernel<D, DT>, (unsigned)(ctas * (PA_ROWS / 32)), 256, 0, 1, true, st, a);
}

// `rows`: query rows per key head that a row of the batch has.
template <int D, int DT>
static cudaError_t launch_attend_few(const AttendArgs& a, int64_t rows, void* ws, cudaStream_t st) {
  if (rows <= 8) {
    // Long contexts take two tiles a step (AtCfg); how long they are only the table's width tells here.
    if constexpr (D == 128) {
      if (((int64_t)a.width << a.bs_shift) >= 1024) return launch_attend<D, DT, 1, 2>(a, ws, st);
    }
    return launch_attend<D, DT, 1>(a, ws, st);
  }
  if constexpr (D < 256) {
    if (rows > 16) return launch_attend<D, DT, 4>(a, ws, st);
  }
  return launch_attend<D, DT, 2>(a, ws, st);
}

// A step of single tokens has `per` query rows per key head and row; else the average decides.  A step with more
// tokens than rows, and enough of them to fill the SMs, may mix prompt chunks, rows of a few tokens and single
// tokens, and only the device knows which is which: rows of pa_from query rows and more go to the tensor-memory
// kernel (which would widen the codes for 256 rows of which `per` are there), the others to the one for few rows, one
// launch after the other on the same workspace.  Its group is that of a single token, or of 16 rows where the average
// row is a short one.  Measured at 64 rows over 50 to 16,000 tokens, 8 key heads of 4 queries of 128 (in groups of 8 for comparison):
// 5 tokens each 512 us (606), 8 tokens 532 (813), 9 tokens 750 (977); tensor memory from 41 rows on, 12 tokens 944 (1,190); single tokens
// beside one chunk of 449 pay for it, 244 (219).  At D = 64 and with more heads per key head the tensor-memory kernel
// is slower than groups of 16 up to 63 rows (9 tokens of D = 64: 668 us, 435).  Steps of chunks alone pay 10 us for the
// second one's empty launches (220 -> 232 us for four chunks of 300 to 400 tokens); 60 single tokens over 6,000 beside two
// chunks of 2,048 take 420 us.
// A step of no more tokens than rows counts as one of single tokens: a chunk among idle rows is right, but goes in
// their groups (200 tokens over 8,000 beside 255 idle rows 213 us, alone 201; 500 beside 511 507 us, alone 171), as the
// launches for chunks would cost every step of single tokens 8 to 10 us.
template <int D, int DT>
static cudaError_t launch_attend_rows(AttendArgs a, void* ws, cudaStream_t st) {
  const int64_t average = (int64_t)a.per * ((a.T + (int64_t)a.B - 1) / a.B);
  a.rows_lo = 0;
  a.rows_hi = INT32_MAX;
  if constexpr (D < 256) {
    if (a.T > a.B && (int64_t)a.heads * a.per * a.T >= (int64_t)PA_ROWS * sm_count(device_index()) / 4) {
      const int pa_from = D == 128 && a.per <= 8 ? 41 : 64;
      a.rows_lo = pa_from;
      const cudaError_t e = launch_attend_tc<D, DT>(a, ws, st);
      if (e != cudaSuccess) return e;
      a.rows_lo = 0;
      a.rows_hi = pa_from;
      return launch_attend_few<D, DT>(a, average < pa_from ? std::max((int64_t)a.per, std::min(average, (int64_t)16)) : a.per, ws, st);
    }
  }
  return launch_attend_few<D, DT>(a, average, ws, st);
}

template <int D>
static cudaError_t launch_attend_dt(int dtype, const AttendArgs& a, void* ws, cudaStream_t st) {
  return dtype == LSS_DTYPE_BF16 ? launch_attend_rows<D, LSS_DTYPE_BF16>(a, ws, st) : launch_attend_rows<D, LSS_DTYPE_F16>(a, ws, st);
}

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
  if ((dtype != LSS_DTYPE_BF16 && dtype != LSS_DTYPE_F16) || T < 0 || heads < 1 || q_heads < heads ||
      q_heads % heads != 0 || !block_size_ok(block_size))
    return LSS_ERR_INVALID_ARG;
  if (q_token_stride < 0 || q_head_stride < 0 || out_token_stride < 0 || out_head_stride < dim) return LSS_ERR_INVALID_ARG;
  if (!table_ok(table, table_stride, width, B, block_size, num_blocks)) return LSS_ERR_INVALID_ARG;
  if (dim != 64 && dim != 128 && dim != 256) return LSS_ERR_UNSUPPORTED;
  if (heads > 65536 || (int64_t)T * q_heads > (1 << 30)) return LSS_ERR_UNSUPPORTED;
  if (B == 0 || T == 0) return LSS_OK;
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
  a.aligned = aligned_to(q, 16) && aligned_to(out, 16) && q_token_stride % 8 == 0 && q_head_stride % 8 == 0 &&
              out_token_stride % 8 == 0 && out_head_stride % 8 == 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  switch (dim) {
    case 64: return status_of(launch_attend_dt<64>(dtype, a, workspace, st));
    case 128: return status_of(launch_attend_dt<128>(dtype, a, workspace, st));
    default: return status_of(launch_attend_dt<256>(dtype, a, workspace, st));
  }
}

}  // extern "C"
