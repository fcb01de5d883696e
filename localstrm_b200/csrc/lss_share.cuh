// lss_share.cuh — blocks of a paged cache that several rows hold: rows that go on from others' tokens,
// and the return of blocks by their last holder.
#pragma once

#include "lss_scan.cuh"

namespace lss {

struct ForkArgs {
  int32_t* table;
  int64_t table_stride;
  int width;
  const int32_t* lens;
  const int32_t* src;   // [n] rows
  const int32_t* dst;
  const int32_t* upto;  // [n] or NULL: tokens taken at most
  int n, B, block_size, num_blocks;
  int32_t* shares;      // [num_blocks]
  const int32_t* free_blocks;
  const int32_t* n_free;
  int32_t* granted;     // [n]
  int32_t* copies;      // [n][2]
  int32_t* lens_out;    // [B], may be lens
  int32_t* n_free_out;  // [1], may be n_free
};

// Which forks are granted, which block each one gets and the new lengths: one CTA, the forks' needs summed up
// in order as the plan's are (lss_plan_kernel).  A row that is named as the destination twice is the first one's.
static __global__ void __launch_bounds__(BL_NT) lss_fork_kernel(ForkArgs a) {
  extern __shared__ int32_t bl_sm[];
  int32_t* claim = bl_sm;  // [B] first fork that names the row as its destination
  __shared__ int64_t scr[32];
  const int tid = threadIdx.x, bs = a.block_size;
  const int nfree = min(max(a.n_free[0], 0), a.num_blocks);
  for (int r = tid; r < a.B; r += BL_NT) claim[r] = INT32_MAX;
  __syncthreads();
  for (int i = tid; i < a.n; i += BL_NT)
    if ((unsigned)a.dst[i] < (unsigned)a.B) atomicMin(&claim[a.dst[i]], i);
  __syncthreads();
  int64_t base = 0;
  int used = 0;
  for (int i0 = 0; i0 < a.n; i0 += BL_NT) {
    const int i = i0 + tid;
    int t = 0, s = 0, d = 0;
    if (i < a.n) {
      s = a.src[i];
      d = a.dst[i];
      if ((unsigned)s < (unsigned)a.B && (unsigned)d < (unsigned)a.B && claim[d] == i && a.lens[d] == 0) {
        t = a.lens[s];
        if (a.upto) t = min(t, a.upto[i]);
        if (t < 0 || t > (int64_t)a.width * bs) t = 0;
      }
    }
    const int need = t % bs != 0;
    int64_t tot;
    const int64_t before = base + bl_scan(need, scr, tot);
    base += tot;
    const bool ok = t > 0 && (need == 0 || before + 1 <= nfree);
    if (i < a.n) {
      int from = -1, to = -1;
      if (ok && need) {
        from = a.table[s * a.table_stride + t / bs];
        to = a.free_blocks[nfree - 1 - before];
        used = (int)before + 1;
        if ((unsigned)to < (unsigned)a.num_blocks) a.shares[to] = 0;
        a.table[d * a.table_stride + t / bs] = to;
      }
      a.copies[2 * i] = from;
      a.copies[2 * i + 1] = to;
      a.granted[i] = ok ? t : 0;
    }
  }
  used = __reduce_max_sync(0xffffffffu, used);
  __syncthreads();
  if ((tid & 31) == 0) scr[tid >> 5] = used;
  __syncthreads();
  used = __reduce_max_sync(0xffffffffu, (int)scr[tid & 31]);
  // All lengths have been read: they may be written in place.
  if (a.lens_out != a.lens)
    for (int r = tid; r < a.B; r += BL_NT) a.lens_out[r] = a.lens[r];
  __syncthreads();
  for (int i = tid; i < a.n; i += BL_NT)
    if (a.granted[i] > 0) a.lens_out[a.dst[i]] = a.granted[i];
  if (tid == 0) a.n_free_out[0] = nfree - used;
}

constexpr int FK_NT = 256;

// The entries of the full blocks from row to row, and a holder more for each: one CTA per fork.
static __global__ void __launch_bounds__(FK_NT) lss_fork_table_kernel(ForkArgs a) {
  pdl_wait();
  const int i = blockIdx.x, full = a.granted[i] / a.block_size;
  if (full == 0) return;
  const int32_t* from = a.table + a.src[i] * a.table_stride;
  int32_t* to = a.table + a.dst[i] * a.table_stride;
  for (int j0 = threadIdx.x; j0 < full; j0 += 4 * FK_NT) {
    int id[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) id[k] = j0 + k * FK_NT < full ? from[j0 + k * FK_NT] : -1;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (j0 + k * FK_NT < full) {
        to[j0 + k * FK_NT] = id[k];
        if ((unsigned)id[k] < (unsigned)a.num_blocks) atomicAdd(&a.shares[id[k]], 1);
      }
  }
}

struct GiveArgs {
  const int32_t* table;
  int64_t table_stride;
  int width;
  const int32_t* lens;
  const int32_t* codes;  // [B] or NULL: none
  const int32_t* keep;   // [B] or NULL: all
  int B, block_size, num_blocks;
  int32_t* shares;       // [num_blocks] or NULL: no block is shared
  int32_t* free_blocks;
  const int32_t* n_free;
  int32_t* lens_out;     // may be lens, or keep
  int32_t* n_free_out;   // may be n_free
  int held;              // pieces of 256 entries that a warp has room for in shared memory
};

constexpr int GV_MARK = -(1 << 30) - 1;  // less the place of a block's last holder: below any count of holders

// Rows with a code give back all of their blocks, the others those behind the tokens they keep; a block goes back on
// the free list with the last of its holders, in the order of these.
//
// shares[block] counts the holders beyond the first.  Every row that gives a block back takes one off (in any
// order: the sum is the same); a count below zero says that nobody holds it any more, and the largest place
// (row * width + entry) among those that gave it takes its place on the list, found by a minimum of GV_MARK - place over
// the count itself.  Then one pass counts per row, and one writes the list and zeroes the counts.  One cluster, a warp
// per row, a cluster barrier between the passes; the rows' numbers of blocks go to all CTAs' shared memory, and the
// entries stay in that of their warp, as far as it goes, so that a pass is one dependent load and not two.  Latency bounds
// it: 512 rows of up to 8,600 tokens in blocks of 16, a third of them stopped: 23 us (on eight SMs 37, and with the table read in every pass 41;
// a quarter of the issue slots, warps wait for fences, cluster barriers and the scattered accesses alike).  Without shares 9 us.
static __global__ void __launch_bounds__(BL_NT) lss_give_kernel(GiveArgs a) {
  extern __shared__ __align__(16) int32_t bl_sm[];
  __shared__ int64_t scr[32];
  cg::cluster_group cl = cg::this_cluster();
  const int rank = (int)cl.block_rank(), nct = (int)cl.num_blocks(), tid = threadIdx.x, lane = tid & 31;
  const int bs = a.block_size, first_row = rank * (BL_NT / 32) + (tid >> 5), step = nct * (BL_NT / 32);
  const int nfree = min(max(a.n_free[0], 0), a.num_blocks);
  // The warp's pieces of 256 entries, in the order of its rows; block, -1 (none), or ~block once it is known to stay out of the list.
  int4* pieces = reinterpret_cast<int4*>(bl_sm) + (size_t)(tid >> 5) * a.held * 64;
  int32_t* upto = bl_sm + (BL_NT / 32) * a.held * 256;  // [B] blocks that go back, then their inclusive sums
  auto kept = [&](int r) {
    const int len = a.lens[r];
    if (a.codes && a.codes[r] != 0) return 0;
    return a.keep ? min(max(a.keep[r], 0), len) : len;
  };
  // Entries [lo, hi) of row r's table.
  auto given = [&](int r, int& lo, int& hi) {
    const int room = a.width * bs;
    lo = blocks_of(min(max(kept(r), 0), room), bs);
    hi = blocks_of(min(max(a.lens[r], 0), room), bs);
  };
  // All rows of the warp, 256 entries at a time: entry k of the lane is j0 + 32 k + lane.  f(row, j0, blocks) may change the
  // blocks that the next pass sees; it returns whether it did.
  auto each = [&](bool fresh, auto begin, auto f, auto finish) {
    int at = 0;
    for (int r = first_row; r < a.B; r += step) {
      int lo, hi;
      given(r, lo, hi);
      begin(r);
      const int32_t* trow = a.table + r * a.table_stride;
      for (int j0 = lo; j0 < hi; j0 += 256, ++at) {
        int id[8];
        const bool room = at < a.held;
        int4* mine = pieces + at * 64 + lane * 2;
        if (!fresh && room) {
          const int4 x = mine[0], y = mine[1];
          id[0] = x.x, id[1] = x.y, id[2] = x.z, id[3] = x.w, id[4] = y.x, id[5] = y.y, id[6] = y.z, id[7] = y.w;
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int j = j0 + 32 * k + lane;
            id[k] = j < hi ? trow[j] : -1;
            if ((unsigned)id[k] >= (unsigned)a.num_blocks) id[k] = -1;
          }
        }
        const bool changed = f(r, j0, id, !fresh && room);
        if ((fresh || changed) && room) {
          mine[0] = make_int4(id[0], id[1], id[2], id[3]);
          mine[1] = make_int4(id[4], id[5], id[6], id[7]);
        }
      }
      finish(r);
    }
  };
  auto nothing = [](int) {};
  if (a.shares) {
    each(true, nothing, [&](int, int, int (&id)[8], bool) {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (id[k] >= 0) atomicSub(&a.shares[id[k]], 1);
      return false;
    }, nothing);
    __threadfence();
    cl.sync();
    each(false, nothing, [&](int r, int j0, int (&id)[8], bool) {
      int left[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) left[k] = id[k] >= 0 ? __ldcg(&a.shares[id[k]]) : 0;
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (left[k] < 0) atomicMin(&a.shares[id[k]], GV_MARK - (r * a.width + j0 + 32 * k + lane));
      return false;
    }, nothing);
    __threadfence();
    cl.sync();
  } else {
    cl.sync();  // every CTA runs: its shared memory may be written
  }
  // Blocks that do not go back with this row are turned to their complement.
  auto choose = [&](int r, int j0, int (&id)[8]) {
    int mark[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) mark[k] = a.shares && id[k] >= 0 ? __ldcg(&a.shares[id[k]]) : 0;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (id[k] >= 0 && a.shares && mark[k] != GV_MARK - (r * a.width + j0 + 32 * k + lane)) id[k] = ~id[k];
  };
  int count = 0;
  each(!a.shares, [&](int) { count = 0; }, [&](int r, int j0, int (&id)[8], bool) {
    choose(r, j0, id);
#pragma unroll
    for (int k = 0; k < 8; ++k) count += id[k] >= 0;
    return true;
  }, [&](int r) {
    const int n = __reduce_add_sync(0xffffffffu, count);
    if (lane < nct) *cl.map_shared_rank(&upto[r], lane) = n;
  });
  cl.sync();
  int64_t base = 0;
  for (int r0 = 0; r0 < a.B; r0 += BL_NT) {
    const int r = r0 + tid;
    const int64_t n = r < a.B ? upto[r] : 0;
    int64_t tot;
    const int64_t first = base + bl_scan(n, scr, tot);
    base += tot;
    if (r < a.B) upto[r] = (int)(first + n);
  }
  __syncthreads();
  int64_t place = 0;
  each(false, [&](int r) { place = (int64_t)nfree + (r > 0 ? upto[r - 1] : 0); }, [&](int r, int j0, int (&id)[8], bool chosen) {
    if (!chosen) choose(r, j0, id);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t vote = __ballot_sync(0xffffffffu, id[k] >= 0);
      if (id[k] >= 0) {
        const int64_t at = place + __popc(vote & ((1u << lane) - 1u));
        if (at < a.num_blocks) a.free_blocks[at] = id[k];
        if (a.shares) a.shares[id[k]] = 0;
      }
      place += __popc(vote);
    }
    return false;
  }, nothing);
  cl.sync();
  if (rank == 0) {
    for (int r = tid; r < a.B; r += BL_NT) a.lens_out[r] = kept(r);
    if (tid == 0) a.n_free_out[0] = (int)min((int64_t)nfree + base, (int64_t)a.num_blocks);
  }
}

}  // namespace lss
