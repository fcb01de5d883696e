// lss_kvmove.cuh — tokens and whole blocks moved inside a paged cache of 8-bit values (e4m3) with one
// scale per block and key head.
#pragma once

#include "lss_kvcache.cuh"

namespace lss {

constexpr int MV_NT = 128;
constexpr int MV_HOLD = 8;  // groups of eight values that a lane holds between reading and writing

struct CompactArgs {
  uint8_t* kc;  // [num_blocks][heads][block_size][dim]
  uint8_t* vc;
  float* ks;    // [num_blocks][heads]
  float* vs;
  int num_blocks, heads, bs_shift, dim;
  const int32_t* table;
  int64_t table_stride;
  int width;
  const int32_t* starts;
  const int32_t* granted;
  const int32_t* lens;
  const int32_t* path;    // [T]
  const int32_t* counts;  // [B]
  int B, T;
};

// e4m3 values times a factor, to nearest even.
__device__ __forceinline__ uint2 mv_scaled(uint2 v, float f) {
  const uint32_t in[4] = {v.x & 0xffffu, v.x >> 16, v.y & 0xffffu, v.y >> 16};
  uint32_t out[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const float2 x = __half22float2(e4m3x2_to_half2((uint16_t)in[q]));
    out[q] = e4m3x2(x.x * f, x.y * f);
  }
  return make_uint2(out[0] | (out[1] << 16), out[2] | (out[3] << 16));
}

// New token path[i] of a row becomes new token i, i < counts[row]: what an accepted branch leaves behind
// the context.  A warp takes a row, a key head, and K or V, block after block.  The scale of a block that takes in
// tokens becomes the largest of those of the blocks that its tokens come from (its own where tokens stay in it), and
// codes of another scale are rounded again, at most by half a step of e4m3 (powers of two: exact down to 2^-6 of the
// scale, where the step stays 2^-9).  As path[i] >= i, blocks and tokens taken in ascending order read nothing that has been
// written; a lane holds what it read over a warp barrier, since other lanes may write there.
// A few hundred bytes per warp: bounded by its chain of dependent loads (lengths, path, table, scale, codes).
static __global__ void __launch_bounds__(MV_NT) lss_compact_kernel(CompactArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * (MV_NT / 32) + (threadIdx.x >> 5);
  const int which = (int)(item % (2 * a.heads)), head = which >> 1;
  const int64_t row = item / (2 * a.heads);
  if (row >= a.B) return;
  const int n = a.granted[row], len = a.lens[row], s = a.starts[row], kept = min(a.counts[row], n);
  if (kept <= 0 || n > len || len > ((int64_t)a.width << a.bs_shift) || s < 0 || (int64_t)s + n > a.T) return;
  const int sh = a.bs_shift, bs = 1 << sh, D = a.dim, d8 = D >> 3;
  const int old = len - n, now = old + kept;
  uint8_t* codes = which & 1 ? a.vc : a.kc;
  float* scales = which & 1 ? a.vs : a.ks;
  const int32_t* path = a.path + s;
  const int32_t* trow = a.table + row * a.table_stride;
  auto source = [&](int i) {  // new token that comes to i: i itself where it is no later one
    const int p = path[i];
    return p > i && p < n ? p : i;
  };
  auto page_of = [&](int pos) {
    const int page = trow[pos >> sh];
    return (unsigned)page < (unsigned)a.num_blocks ? page : -1;
  };
  for (int j = old >> sh; j <= (now - 1) >> sh; ++j) {
    const int i0 = max((j << sh) - old, 0), i1 = min(((j + 1) << sh) - old, kept);
    const int page = page_of(j << sh);
    if (page < 0) continue;
    // Does anything move, and from which scales?
    bool moves = false;
    float top = 0.0f;
    for (int i = i0 + lane; i < i1; i += 32) {
      const int p = source(i), from = page_of(old + p);
      if (p != i && from >= 0) {
        moves = true;
        top = fmaxf(top, scales[(int64_t)from * a.heads + head]);
      }
    }
    if (!__any_sync(0xffffffffu, moves)) continue;
    float* at = scales + (int64_t)page * a.heads + head;
    const float was = *at;
    bool stays = (j << sh) < old;
    for (int i = i0 + lane; i < i1; i += 32) {
      const int p = source(i);
      stays |= p == i || page_of(old + p) < 0;
    }
    if (__any_sync(0xffffffffu, stays)) top = fmaxf(top, was);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    uint8_t* dst = codes + (((int64_t)page * a.heads + head) << sh) * D;
    // Groups of eight values of the tokens of this block that stay (where its scale changes) or come.
    const int lo = top != was ? 0 : max(old - (j << sh), 0), hi = min(now - (j << sh), bs);
    const int e1 = hi * d8;
    for (int e0 = lo * d8; e0 < e1; e0 += 32 * MV_HOLD) {
      uint2 hold[MV_HOLD];
      float f[MV_HOLD];
#pragma unroll
      for (int k = 0; k < MV_HOLD; ++k) {
        const int e = e0 + 32 * k + lane;
        f[k] = 0.0f;
        if (e < e1) {
          const int t = e / d8, i = (j << sh) + t - old, c = e - t * d8;
          const int p = i >= 0 ? source(i) : i, pos = old + p;
          int from = p != i ? page_of(pos) : page, off = pos & (bs - 1);
          if (from < 0) {  // nothing to read: what is here stays
            from = page;
            off = t;
          }
          const int64_t ph = (int64_t)from * a.heads + head;
          const float own = from == page ? was : scales[ph];
          f[k] = own == top ? 1.0f : __fdiv_rn(own, top);  // all scales 0, in a caller's own cache: the codes as they are
          hold[k] = *reinterpret_cast<const uint2*>(codes + ((ph << sh) + off) * D + c * 8);
        }
      }
      __syncwarp();
#pragma unroll
      for (int k = 0; k < MV_HOLD; ++k) {
        const int e = e0 + 32 * k + lane;
        if (e < e1) *reinterpret_cast<uint2*>(dst + e * 8) = f[k] == 1.0f ? hold[k] : mv_scaled(hold[k], f[k]);
      }
      __syncwarp();
    }
    if (lane == 0 && top != was) *at = top;
    __syncwarp();
  }
}

struct CopyArgs {
  uint8_t* kc;
  uint8_t* vc;
  float* ks;
  float* vs;
  int num_blocks, heads;
  int64_t pieces;          // 16-byte pieces of a block
  const int32_t* copies;   // [n][2]: from, to
  int n, parts;            // CTAs per block of K or V
};

constexpr int CP_NT = 256, CP_PER = 4;  // 16 KB per CTA

// Whole blocks with their scales, from copies[i][0] to copies[i][1]; pairs that are not two blocks of the
// cache are passed over.  Bound by HBM, or by its two dependent loads where there is little to copy.
static __global__ void __launch_bounds__(CP_NT) lss_copy_kernel(CopyArgs a) {
  const int part = (int)(blockIdx.x % a.parts), rest = (int)(blockIdx.x / a.parts), i = rest >> 1;
  const int from = a.copies[2 * i], to = a.copies[2 * i + 1];
  if ((unsigned)from >= (unsigned)a.num_blocks || (unsigned)to >= (unsigned)a.num_blocks || from == to) return;
  uint4* codes = reinterpret_cast<uint4*>(rest & 1 ? a.vc : a.kc);
  const uint4* src = codes + from * a.pieces;
  uint4* dst = codes + to * a.pieces;
  const int64_t p0 = (int64_t)part * (CP_NT * CP_PER) + threadIdx.x;
  uint4 v[CP_PER];
#pragma unroll
  for (int k = 0; k < CP_PER; ++k)
    if (p0 + k * CP_NT < a.pieces) v[k] = src[p0 + k * CP_NT];
  if (part == 0) {
    float* scales = rest & 1 ? a.vs : a.ks;
    for (int h = threadIdx.x; h < a.heads; h += CP_NT) scales[(int64_t)to * a.heads + h] = scales[(int64_t)from * a.heads + h];
  }
#pragma unroll
  for (int k = 0; k < CP_PER; ++k)
    if (p0 + k * CP_NT < a.pieces) dst[p0 + k * CP_NT] = v[k];
}

}  // namespace lss
