// lss_blocks.cuh — block tables and slot maps of a paged key/value cache, built from the
// requests' lengths on the device, and the return of stopped requests' blocks.
#pragma once

#include "lss_scan.cuh"

namespace lss {

struct PlanArgs {
  int32_t* table;  // [B][table_stride], `width` entries used
  int64_t table_stride;
  int width;
  const int32_t* lens;
  const int32_t* new_lens;
  int B, block_size, num_blocks, capacity;
  const int32_t* free_blocks;  // a stack: the next block is free_blocks[n_free - 1]
  const int32_t* n_free;
  int64_t* slots;       // [capacity]
  int32_t* positions;   // [capacity]
  int32_t* starts;      // [B + 1]
  int32_t* granted;     // [B]
  int32_t* lens_out;    // [B], may be lens
  int32_t* n_free_out;  // [1], may be n_free
};

// One step's plan.  With new = max(new_lens, 0), upto the inclusive sums of new and
// need = ceil((len + new) / bs) - ceil(len / bs) for the rows whose tokens fit (the capacity and
// the table's width, else 0), a row is granted if the inclusive sum of need is within the free
// list (or it needs no block): rows are served in order, and the k-th block taken is
// free_blocks[n_free - 1 - k].
//
// The work is a few hundred kilobytes at most: what bounds it is the chain load lengths -> two
// block-wide sums -> a search and two dependent loads per token, not bytes.  So it is one launch: every CTA
// takes the sums of all rows by itself (cheaper than passing them on through memory and a second
// launch), and each fills its share of the tokens.  Where the new state is written in place the CTAs are one
// cluster, with a barrier between the last read of the lengths and their update; else there are as many as the
// tokens need (65,000 tokens of 1,000 rows: eight CTAs issue for 14 us, 64 for 5).
__global__ void __launch_bounds__(BL_NT) lss_plan_kernel(PlanArgs a) {
  extern __shared__ int32_t bl_sm[];
  int32_t* upto = bl_sm;          // [B] inclusive sums of the new tokens, at most INT_MAX
  int32_t* taken = bl_sm + a.B;   // [B] blocks taken by the rows before, -1: not granted
  __shared__ int64_t scr[32];
  cg::cluster_group cl = cg::this_cluster();
  const int rank = blockIdx.x, nct = gridDim.x, tid = threadIdx.x;
  const int bs = a.block_size;
  const int nfree = min(max(a.n_free[0], 0), a.num_blocks);
  int64_t base_tok = 0, base_need = 0;
  int used = 0;  // blocks that granted rows of this thread and the ones before them take
  for (int r0 = 0; r0 < a.B; r0 += BL_NT) {
    const int r = r0 + tid;
    const bool in = r < a.B;
    const int64_t len = in ? a.lens[r] : 0;
    const int64_t nw = in ? max(a.new_lens[r], 0) : 0;
    int64_t tot;
    const int64_t first = base_tok + bl_scan(nw, scr, tot);
    base_tok += tot;
    const bool fits = nw > 0 && len >= 0 && first + nw <= a.capacity && len + nw <= (int64_t)a.width * bs;
    const int64_t need = fits ? blocks_of((int)(len + nw), bs) - blocks_of((int)len, bs) : 0;
    const int64_t before = base_need + bl_scan(need, scr, tot);
    base_need += tot;
    const bool ok = fits && (need == 0 || before + need <= nfree);
    if (in) {
      upto[r] = (int)min(first + nw, (int64_t)INT32_MAX);
      taken[r] = ok ? (int)min(before, (int64_t)nfree) : -1;
      if (ok && need > 0) used = (int)(before + need);
      if (rank == 0) {
        a.starts[r] = (int)min(first, (int64_t)a.capacity);
        a.granted[r] = ok ? (int)nw : 0;
        if (r == a.B - 1) a.starts[a.B] = (int)min(first + nw, (int64_t)a.capacity);
      }
    }
  }
  if (a.B == 0 && rank == 0 && tid == 0) a.starts[0] = 0;
  // Largest `used` of all threads: sums of the needs only grow, so it belongs to the last granted row.
  used = __reduce_max_sync(0xffffffffu, used);
  __syncthreads();
  if ((tid & 31) == 0) scr[tid >> 5] = used;
  __syncthreads();
  used = __reduce_max_sync(0xffffffffu, (int)scr[tid & 31]);

  const int total = (int)min(base_tok, (int64_t)a.capacity);
  // Four tokens a thread at a time: their searches and loads run side by side.
  constexpr int TOK = 4;
  const int64_t stride = (int64_t)nct * BL_NT;
  for (int64_t t0 = (int64_t)rank * BL_NT + tid; t0 < a.capacity; t0 += TOK * stride) {
    int row[TOK], page[TOK], pos[TOK], off[TOK];
    int32_t* entry[TOK];
    bool fresh[TOK];
#pragma unroll
    for (int i = 0; i < TOK; ++i) {
      const int64_t t = t0 + i * stride;
      int lo = 0, hi = t < total ? a.B - 1 : 0;  // first row whose sum exceeds t
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (upto[mid] > t) hi = mid; else lo = mid + 1;
      }
      row[i] = t < total ? lo : -1;
    }
#pragma unroll
    for (int i = 0; i < TOK; ++i) {
      const int r = row[i];
      pos[i] = off[i] = 0;
      page[i] = -1;
      entry[i] = nullptr;
      fresh[i] = false;
      if (r >= 0) {
        const int len = a.lens[r], tk = taken[r];
        const int64_t p = (int64_t)len + t0 + i * stride - (r > 0 ? upto[r - 1] : 0);
        pos[i] = (int)p;
        if (tk >= 0) {
          const int j = (int)((unsigned)p / (unsigned)bs), held = blocks_of(len, bs);
          off[i] = (int)p - j * bs;
          entry[i] = a.table + r * a.table_stride + j;
          fresh[i] = j >= held;
          page[i] = fresh[i] ? a.free_blocks[nfree - 1 - (tk + j - held)] : *entry[i];
        }
      }
    }
#pragma unroll
    for (int i = 0; i < TOK; ++i) {
      const int64_t t = t0 + i * stride;
      if (t < a.capacity) {
        if (fresh[i] && off[i] == 0) *entry[i] = page[i];  // a block taken now starts with a token of this step
        a.slots[t] = page[i] >= 0 && page[i] < a.num_blocks ? (int64_t)page[i] * bs + off[i] : -1;
        a.positions[t] = pos[i];
      }
    }
  }
  // In place, the grid is one cluster: every CTA has read the lengths and the free count, the first one may
  // write over them.
  cl.sync();
  if (rank == 0) {
    for (int r = tid; r < a.B; r += BL_NT) {
      const int nw = max(a.new_lens[r], 0);
      a.lens_out[r] = a.lens[r] + (taken[r] >= 0 ? nw : 0);
    }
    if (tid == 0) a.n_free_out[0] = nfree - used;
  }
}

struct ReleaseArgs {
  const int32_t* table;
  int64_t table_stride;
  int width;
  const int32_t* lens;
  const int32_t* codes;
  int B, block_size, num_blocks;
  int32_t* free_blocks;
  const int32_t* n_free;
  int32_t* lens_out;    // may be lens
  int32_t* n_free_out;  // may be n_free
};

// The blocks of the rows with a non-zero code go back on the free list, in row and block order,
// and their lengths become 0.  Same shape as the plan: sums of all rows in every CTA, then one warp
// per stopped row copies its table entries (contiguous on both sides).
__global__ void __launch_bounds__(BL_NT) lss_release_kernel(ReleaseArgs a) {
  extern __shared__ int32_t bl_sm[];
  int32_t* upto = bl_sm;  // [B] inclusive sums of the blocks given back, at most INT_MAX
  __shared__ int64_t scr[32];
  cg::cluster_group cl = cg::this_cluster();
  const int rank = (int)cl.block_rank(), nct = (int)cl.num_blocks(), tid = threadIdx.x;
  const int bs = a.block_size;
  const int nfree = min(max(a.n_free[0], 0), a.num_blocks);
  int64_t base = 0;
  for (int r0 = 0; r0 < a.B; r0 += BL_NT) {
    const int r = r0 + tid;
    int64_t n = 0;
    if (r < a.B && a.codes[r] != 0)
      n = blocks_of(min(max(a.lens[r], 0), a.width * bs), bs);
    int64_t tot;
    const int64_t first = base + bl_scan(n, scr, tot);
    base += tot;
    if (r < a.B) upto[r] = (int)min(first + n, (int64_t)INT32_MAX);
  }
  __syncthreads();
  const int lane = tid & 31;
  for (int r = rank * (BL_NT / 32) + (tid >> 5); r < a.B; r += nct * (BL_NT / 32)) {
    const int first = r > 0 ? upto[r - 1] : 0, n = upto[r] - first;
    for (int j0 = lane; j0 < n; j0 += 32 * 8) {  // eight loads on their way before the first store
      int32_t ids[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) ids[i] = j0 + 32 * i < n ? a.table[r * a.table_stride + j0 + 32 * i] : 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int64_t at = (int64_t)nfree + first + j0 + 32 * i;
        if (j0 + 32 * i < n && at < a.num_blocks) a.free_blocks[at] = ids[i];
      }
    }
  }
  cl.sync();
  if (rank == 0) {
    for (int r = tid; r < a.B; r += BL_NT) a.lens_out[r] = a.codes[r] != 0 ? 0 : a.lens[r];
    if (tid == 0) a.n_free_out[0] = (int)min((int64_t)nfree + base, (int64_t)a.num_blocks);
  }
}

}  // namespace lss
