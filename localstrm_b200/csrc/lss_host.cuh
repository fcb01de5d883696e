// lss_host.cuh — what the C entries of the decode-step operators share: device queries, launches and
// checks of pointers and sizes.
#pragma once

#include <algorithm>
#include <cstdlib>
#include <mutex>
#include <utility>

#include "lss_common.cuh"

using namespace lss;

static constexpr int MAX_DEV = 64;

static inline int device_index() {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= MAX_DEV) dev = 0;
  return dev;
}

static std::mutex g_mu;

static inline int sm_count(int dev) {
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
static inline cudaError_t allow_smem(K kern, SmemSet& set, int dev, int bytes) {
  std::lock_guard<std::mutex> lock(g_mu);
  if (bytes <= set.bytes[dev]) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) set.bytes[dev] = bytes;
  return e;
}

template <class... KA, class... A>
static inline cudaError_t launch(void (*kern)(KA...), unsigned grid, unsigned block, size_t smem, int cluster, bool pdl,
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

static inline int status_of(cudaError_t e) {
  if (e == cudaSuccess) return LSS_OK;
  cudaGetLastError();
  return LSS_ERR_CUDA;
}

static inline bool aligned_to(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
static inline bool known_dtype(int d) { return d == LSS_DTYPE_F32 || d == LSS_DTYPE_BF16 || d == LSS_DTYPE_F16; }
static inline bool block_size_ok(int bs) { return bs == 16 || bs == 32 || bs == 64 || bs == 128 || bs == 256; }
// Rows of two matrices (start, bytes between rows, bytes of a row) that share memory.  Rows of one pitch may lie
// beside each other.
static inline bool rows_overlap(const void* x, int64_t x_pitch, int64_t x_row, const void* y, int64_t y_pitch, int64_t y_row, int rows) {
  const int64_t d = (int64_t)(reinterpret_cast<intptr_t>(y) - reinterpret_cast<intptr_t>(x));
  if (d >= (rows - 1) * x_pitch + x_row || -d >= (rows - 1) * y_pitch + y_row) return false;
  if (rows == 1 || x_pitch != y_pitch) return true;
  const int64_t at = (d % x_pitch + x_pitch) % x_pitch;  // where y's rows start in x's pitch
  return at < x_row || at + y_row > x_pitch;
}
// Two arrays of rows of n bytes with equal strides st and sh, the second one d bytes behind the first, of which two rows share
// memory: rows i and j strides apart begin d + i st + j sh bytes apart, i among Tx and Ty, j among Hx and Hy of them.
static inline bool rows_meet(int64_t d, int64_t st, int64_t sh, int64_t Tx, int64_t Ty, int64_t Hx, int64_t Hy, int64_t n) {
  if (Tx + Ty < Hx + Hy) {  // the walk is over the shorter side
    std::swap(Tx, Hx);
    std::swap(Ty, Hy);
    std::swap(st, sh);
  }
  for (int64_t j = 1 - Hx; j < Hy; ++j) {
    const int64_t r = d + j * sh, i0 = st > 0 ? (r >= 0 ? -((r + st - 1) / st) : -r / st) : 0;  // r + i0 st <= 0 < r + (i0 + 1) st
    for (int64_t i = i0; i <= i0 + 1; ++i)  // the nearest ones that there are
      if (std::abs(r + std::min(std::max(i, 1 - Tx), Ty - 1) * st) < n) return true;
  }
  return false;
}
// Two arrays of T x H rows of n bytes (start, bytes between tokens and between heads) that share memory without
// being the same rows: a result would be written where another CTA still reads its query.  With equal strides
// exactly, else wherever the extents meet.
static inline bool rows_shifted(const void* x, int64_t x_st, int64_t x_sh, const void* y, int64_t y_st, int64_t y_sh, int64_t T, int64_t H, int64_t n) {
  if (T == 1) x_st = y_st = 0;  // one token, one head: the stride says nothing
  if (H == 1) x_sh = y_sh = 0;
  const int64_t d = (int64_t)(reinterpret_cast<intptr_t>(y) - reinterpret_cast<intptr_t>(x));
  if (d >= (T - 1) * x_st + (H - 1) * x_sh + n || -d >= (T - 1) * y_st + (H - 1) * y_sh + n) return false;
  if (x_st != y_st || x_sh != y_sh) return true;
  return d != 0 && rows_meet(d, x_st, x_sh, T, T, H, H, n);
}
// Arrays of n entries of which one begins inside the other.
static inline bool cut(const int32_t* x, const int32_t* y, int64_t n) { return x != y && x < y + n && y < x + n; }
static inline int log2_of(int v) {
  int s = 0;
  while ((1 << s) < v) ++s;
  return s;
}
static inline int cluster_for(int64_t ctas, int most) {
  int c = 1;
  while (c < most && c < ctas) c <<= 1;
  return c;
}

// ---------------------------------------------------------------- block tables
static inline bool table_ok(const void* table, int64_t stride, int width, int B, int bs, int num_blocks) {
  return (table || B == 0) && width >= 1 && stride >= width && B >= 0 && bs >= 1 && num_blocks >= 1 &&
         (int64_t)width * bs <= (1 << 30);
}
