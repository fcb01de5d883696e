// lss_tree.cuh — the trees of a step's drafted tokens, and which of them the sampled tokens accept.
#pragma once

#include "lss_scan.cuh"

namespace lss {

constexpr int TR_NT = 128;                   // threads of a row's CTA
constexpr int TR_MOST = LSS_TREE_MAX_TOKENS; // longest row whose parents are read
constexpr int TR_PER = TR_MOST / TR_NT;
constexpr int AC_NT = 128;

struct TreeArgs {
  const int32_t* starts;   // [B + 1]
  const int32_t* granted;  // [B]
  const int32_t* lens;     // [B]
  const int32_t* parents;  // [T]
  int2* span;              // [T]
  int32_t* positions;      // [T]
  int B, T;
};

// New tokens of row b (0: none, or numbers that do not fit), and where its part of the step's tokens ends.
__device__ __forceinline__ int tr_row(const int32_t* starts, const int32_t* granted, const int32_t* lens, int b, int T, int& s, int& end) {
  s = min(max(starts[b], 0), T);
  end = min(max(starts[b + 1], s), T);
  const int n = granted[b];
  return n > 0 && n <= lens[b] && starts[b] == s && (int64_t)s + n <= T ? n : 0;
}
// Parent of new token i of n: none (-1) where what is given is no earlier one; the token before in rows too long to be trees.
__device__ __forceinline__ int tr_parent(const int32_t* parents, int i, int n) {
  if (n > TR_MOST) return i - 1;
  const int p = parents[i];
  return p >= 0 && p < i ? p : -1;
}

// For each token its place in the pre-order of its row's forest (children in order), the size of its
// branch and its position, context + depth: token j is an ancestor of i, or i itself, where
//   0 <= place(i) - place(j) < size(j).
// One CTA per row; all sums go along the parents by doubling, in log2(depth) rounds over shared memory:
//   size: tokens at distance < 2^k below a node, to which those of the nodes 2^k below it are added;
//   depth and place: sums over the ancestors of 1 and of (1 + sizes of the earlier children of the same parent).
// A chain (every token follows the one before) is written as it is.  Nothing here is more than a
// few kilobytes per row; latency bounds it.
static __global__ void __launch_bounds__(TR_NT) lss_tree_kernel(TreeArgs a) {
  __shared__ int par[TR_MOST], size[TR_MOST], sum[TR_MOST], jump[TR_MOST];
  const int b = blockIdx.x, tid = threadIdx.x;
  if (b == a.B) {  // tokens before the first row and behind the last one
    const int first = a.B > 0 ? min(max(a.starts[0], 0), a.T) : 0, last = a.B > 0 ? min(max(a.starts[a.B], 0), a.T) : 0;
    for (int i = tid; i < a.T; i += TR_NT)
      if (i < first || i >= last) {
        a.span[i] = make_int2(0, 0);
        a.positions[i] = 0;
      }
    return;
  }
  int s, end;
  const int n = tr_row(a.starts, a.granted, a.lens, b, a.T, s, end);
  for (int i = s + n + tid; i < end; i += TR_NT) {
    a.span[i] = make_int2(0, 0);
    a.positions[i] = 0;
  }
  if (n == 0) return;
  const int ctx = a.lens[b] - n;
  bool chain = true;
  for (int i = tid; i < n && n <= TR_MOST; i += TR_NT) {
    const int p = tr_parent(a.parents + s, i, n);
    par[i] = jump[i] = p;
    size[i] = 1;
    chain = chain && p == i - 1;
  }
  if (__syncthreads_and(chain)) {
    for (int i = tid; i < n; i += TR_NT) {
      a.span[s + i] = make_int2(i, n - i);
      a.positions[s + i] = ctx + i;
    }
    return;
  }
  const int per = (n + TR_NT - 1) / TR_NT;
  // Sizes.
  for (;;) {
    int up[TR_PER], up2[TR_PER], have[TR_PER];
    bool more = false;
#pragma unroll
    for (int k = 0; k < TR_PER; ++k) {
      const int i = tid + k * TR_NT;
      up[k] = up2[k] = -1;
      if (k < per && i < n) {
        up[k] = jump[i];
        have[k] = size[i];
        if (up[k] >= 0) up2[k] = jump[up[k]];
        more |= up2[k] >= 0;
      }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < TR_PER; ++k) {
      const int i = tid + k * TR_NT;
      if (k < per && i < n) {
        if (up[k] >= 0) atomicAdd(&size[up[k]], have[k]);
        jump[i] = up2[k];
      }
    }
    if (!__syncthreads_or(more)) break;
  }
  // Sizes of the earlier children of the same parent; they lie between the parent and the token.
  for (int k = 0; k < per; ++k) {
    const int i = tid + k * TR_NT;
    if (i >= n) break;
    const int p = par[i];
    int before = 1;
    for (int j = p + 1; j < i; ++j)
      if (par[j] == p) before += size[j];
    sum[i] = before | (1 << 16);  // the depth in the upper half
    jump[i] = p;
  }
  __syncthreads();
  for (;;) {
    int up[TR_PER], up2[TR_PER], add[TR_PER];
    bool more = false;
#pragma unroll
    for (int k = 0; k < TR_PER; ++k) {
      const int i = tid + k * TR_NT;
      up[k] = up2[k] = -1;
      add[k] = 0;
      if (k < per && i < n) {
        up[k] = jump[i];
        if (up[k] >= 0) {
          add[k] = sum[up[k]];
          up2[k] = jump[up[k]];
        }
        more |= up2[k] >= 0;
      }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < TR_PER; ++k) {
      const int i = tid + k * TR_NT;
      if (k < per && i < n) {
        sum[i] += add[k];
        jump[i] = up2[k];
      }
    }
    if (!__syncthreads_or(more)) break;
  }
  for (int i = tid; i < n; i += TR_NT) {
    a.span[s + i] = make_int2((sum[i] & 0xffff) - 1, size[i]);
    a.positions[s + i] = ctx + (sum[i] >> 16) - 1;
  }
}

struct AcceptArgs {
  const int32_t* starts;
  const int32_t* granted;
  const int32_t* lens;
  const int32_t* parents;  // [T]
  const int32_t* drafts;   // [T]
  const int32_t* targets;  // [T]
  const int32_t* codes;    // [T] or NULL
  const int32_t* given;    // [B] or NULL: 1
  int32_t* path;           // [T]
  int32_t* tokens;         // [T]
  int32_t* counts;         // [B]
  int32_t* lens_out;       // [B], may be lens
  int32_t* last;           // [B]
  int32_t* codes_out;      // [B]
  int B, T;
};

// A warp per row.  The first `given` tokens are accepted as they are; from the last of them the walk goes on to
// the first child that is the token sampled at its parent, until there is none or the sampled token has a stop code.
// The first 64 tokens of a row stay in registers, two per lane: a step is two votes and a few shuffles; what lies behind
// them is read as it is needed.
static __global__ void __launch_bounds__(AC_NT) lss_accept_kernel(AcceptArgs a) {
  const int lane = threadIdx.x & 31, b = blockIdx.x * (AC_NT / 32) + (threadIdx.x >> 5);
  if (b > a.B) return;
  if (b == a.B) {
    const int first = a.B > 0 ? min(max(a.starts[0], 0), a.T) : 0, last = a.B > 0 ? min(max(a.starts[a.B], 0), a.T) : 0;
    for (int i = lane; i < a.T; i += 32)
      if (i < first || i >= last) a.path[i] = a.tokens[i] = -1;
    return;
  }
  int s, end;
  const int n = tr_row(a.starts, a.granted, a.lens, b, a.T, s, end), len = a.lens[b];
  for (int i = s + n + lane; i < end; i += 32) a.path[i] = a.tokens[i] = -1;
  if (n == 0) {
    if (lane == 0) {
      a.counts[b] = a.codes_out[b] = 0;
      a.last[b] = -1;
      a.lens_out[b] = len - max(a.granted[b], 0);
    }
    return;
  }
  const int32_t *par = a.parents + s, *dr = a.drafts + s, *tg = a.targets + s, *cd = a.codes ? a.codes + s : nullptr;
  int p[2], d[2], t[2], c[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int i = lane + 32 * k;
    const bool in = i < n;
    p[k] = in ? tr_parent(par, i, n) : -2;
    d[k] = in ? dr[i] : 0;
    t[k] = in ? tg[i] : 0;
    c[k] = in && cd ? cd[i] : 0;
  }
  auto at = [&](const int (&r)[2], const int32_t* from, int i) {  // one token's number, the same for all lanes
    if (i >= 64) return from[i];
    const int x = __shfl_sync(0xffffffffu, r[0], i & 31), y = __shfl_sync(0xffffffffu, r[1], i & 31);
    return i < 32 ? x : y;
  };
  const int given = min(max(a.given ? a.given[b] : 1, 1), n);
  for (int i = lane; i < given; i += 32) a.path[s + i] = i;
  int cur = given - 1, count = given, said = 0, target, code;
  for (;;) {
    target = at(t, tg, cur);
    code = cd ? at(c, cd, cur) : 0;
    if (lane == 0) a.tokens[s + said] = target;
    ++said;
    if (code != 0) break;
    int next = -1;
    const uint32_t hit0 = __ballot_sync(0xffffffffu, p[0] == cur && d[0] == target);
    const uint32_t hit1 = __ballot_sync(0xffffffffu, p[1] == cur && d[1] == target);
    if (hit0) {
      next = __ffs(hit0) - 1;
    } else if (hit1) {
      next = 32 + __ffs(hit1) - 1;
    } else {
      for (int i0 = max(64, cur + 1) & ~31; i0 < n && next < 0; i0 += 32) {
        const int i = i0 + lane;
        const uint32_t hit = __ballot_sync(0xffffffffu, i < n && tr_parent(par, i, n) == cur && dr[i] == target);
        if (hit) next = i0 + __ffs(hit) - 1;
      }
    }
    if (next < 0) break;
    if (lane == 0) a.path[s + count] = next;
    ++count;
    cur = next;
  }
  for (int i = count + lane; i < n; i += 32) a.path[s + i] = -1;
  for (int i = said + lane; i < n; i += 32) a.tokens[s + i] = -1;
  if (lane == 0) {
    a.counts[b] = count;
    a.lens_out[b] = len - n + count;
    a.last[b] = target;
    a.codes_out[b] = code;
  }
}

}  // namespace lss
