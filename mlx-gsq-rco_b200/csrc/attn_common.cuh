// What the kernels of attention over the quantised cache share: arguments,
// the sequences' lengths and the order of their work, dequantisation.
#pragma once

#include "gsq_common.cuh"
#include "gsq_kv.h"
#include "kv_codes.cuh"

namespace gsq {

struct AttnArgs {
  const void* q;
  int64_t qb, qn, qh;  // strides in elements (sequence, token, head)
  const uint8_t *kc, *vc;
  const float *ks, *vs;
  int batch, n, heads, kv, group, dim;
  int64_t cap;
  const int32_t* start;
  int64_t start_stride;
  const int32_t* counts;
  const int32_t* tree;
  int64_t tree_stride;
  int words;  // of a tree's row
  const float* gate;
  int64_t gb, gn, gh;
  float scale;
  void* out;
  int ctas, rows8;      // CTAs of the split, rows of a partial result
  int* err;             // device error word
  float *part, *stat;   // [2 * ctas][rows8][dim], [2 * ctas][rows8][2] (max in base 2, sum)
  struct Joint* joints;  // [ctas], for the joining launch
  int cluster, blocks;   // token kernel by units: CTAs per unit, units (of 16 rows each, or 8) per key/value head
  int joins;             // CTAs that join one unit's parts (row-block kernel)
};

// Cached positions and new tokens of sequence b. Caches hold at most 2^30 positions, so a start past that sees all of
// them as cached text, and one below -2^29 leaves no row anything (n <= 65536): within these bounds an int holds
// every sum and difference of positions.
struct SeqSpan {
  int base;   // position of the first new token
  int count;  // new tokens (0: all rows are padding)
  int len;    // positions that any of them may see, from 0
};

__device__ __forceinline__ SeqSpan seq_span(const AttnArgs& a, int b) {
  SeqSpan s;
  s.base = min(max(a.start[(int64_t)b * a.start_stride], -(1 << 29)), 1 << 30);
  s.count = a.counts ? min(max(a.counts[b], 0), a.n) : a.n;
  s.len = s.count > 0 ? min(max(s.base + s.count, 0), (int)a.cap) : 0;
  return s;
}

// The work is a list of tiles of positions, ordered by sequence, key/value head, block of rows (one, where all rows
// of a head are taken together) and position; a unit is the tiles of one (sequence, head, block). CTA c of G takes
// tiles [c T / G, (c + 1) T / G), where G is at most T: no CTA below G is without a tile, so the parts of a unit are
// those of consecutive CTAs. Every warp finds its place by itself, 32 sequences at a time, one per lane.
struct Place {
  int b, kh, mb;    // unit
  int tile, tiles;  // tile in it, and its tiles
  SeqSpan span;
};

// A unit in several CTAs' parts, noted by the second of them (c0 + 1): part of CTA c0 in slot s0, of c0 + 1 .. c1 in
// slots 2 c. parts == 0: CTA c does not begin in a unit's second part.
struct Joint {
  int parts, b, kh, mb, c0, s0, count, pad;
  // Slot of part i among the partial results.
  __device__ int slot(int i) const { return i == 0 ? s0 : 2 * (c0 + i); }
};

// Shape: blocks(a) row blocks of ROWS rows each; tiles(a, span, mb).
template <typename Shape>
struct TileList {
  // Tiles of one head of sequence b.
  __device__ static int of_head(const AttnArgs& a, int b) {
    if (b >= a.batch) return 0;
    const SeqSpan s = seq_span(a, b);
    int sum = 0;
    for (int mb = 0; mb < Shape::blocks(a); mb++) sum += Shape::tiles(a, s, mb);
    return sum;
  }
  __device__ static int total(const AttnArgs& a) {
    int s = 0;
    const int blocks = Shape::blocks(a), pairs = a.batch * blocks;
    for (int i = threadIdx.x & 31; i < pairs; i += 32) s += Shape::tiles(a, seq_span(a, i / blocks), i % blocks);
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s * a.kv;
  }
  // Where tile t (below the total) lies; every lane of the warp calls it. The lanes take a sequence each, or where a
  // head has many blocks a block each of one sequence after the other.
  __device__ static Place locate(const AttnArgs& a, int t) {
    const int lane = threadIdx.x & 31, blocks = Shape::blocks(a);
    Place p = {};
    auto scan = [&](int v) {
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
      }
      return v;
    };
    int done = 0, head = 0;
    if (blocks <= 4) {
      for (int b0 = 0; b0 < a.batch; b0 += 32) {
        const int mine = of_head(a, b0 + lane) * a.kv;
        const int sum = scan(mine);
        const unsigned past = __ballot_sync(0xffffffffu, t < done + sum);
        if (past) {
          const int l = __ffs(past) - 1;
          done += __shfl_sync(0xffffffffu, sum - mine, l);
          head = __shfl_sync(0xffffffffu, mine, l) / a.kv;
          p.b = b0 + l;
          break;
        }
        done += __shfl_sync(0xffffffffu, sum, 31);
      }
    } else {
      for (;; p.b++) {
        const SeqSpan span = seq_span(a, p.b);
        head = 0;
        for (int mb = lane; mb < blocks; mb += 32) head += Shape::tiles(a, span, mb);
        head = __reduce_add_sync(0xffffffffu, head);
        if (t < done + head * a.kv) break;
        done += head * a.kv;
      }
    }
    p.kh = (t - done) / head;
    p.tile = (t - done) % head;
    p.span = seq_span(a, p.b);
    for (;; p.mb += 32) {
      const int mine = p.mb + lane < blocks ? Shape::tiles(a, p.span, p.mb + lane) : 0;
      const int sum = scan(mine);
      const unsigned past = __ballot_sync(0xffffffffu, p.tile < sum);
      if (past) {
        const int l = __ffs(past) - 1;
        p.tile -= __shfl_sync(0xffffffffu, sum - mine, l);
        p.tiles = __shfl_sync(0xffffffffu, mine, l);
        p.mb += l;
        return p;
      }
      p.tile -= __shfl_sync(0xffffffffu, sum, 31);
    }
  }
  // What the joining launch has to know of CTA c, which begins with tile t at p (one thread): the unit, if c is the
  // second that has a part of it.
  __device__ static void note(const AttnArgs& a, int c, int t, const Place& p, int total, int ctas) {
    Joint j = {};
    const int t0 = t - p.tile;
    j.c0 = cta_of(t0, total, ctas);
    if (p.tile && j.c0 == c - 1) {
      j.parts = cta_of(t0 + p.tiles - 1, total, ctas) - j.c0 + 1;
      j.b = p.b;
      j.kh = p.kh;
      j.mb = p.mb;
      j.s0 = 2 * j.c0 + (first_of(j.c0, total, ctas) == t0 ? 0 : 1);  // CTA c0 may have begun another unit before it
      j.count = p.span.count;
    }
    a.joints[c] = j;
  }
  // The first tile of the unit after p's; there must be one.
  __device__ static void next_unit(const AttnArgs& a, Place& p) {
    p.tile = 0;
    do {
      if (++p.mb == Shape::blocks(a)) {
        p.mb = 0;
        if (++p.kh == a.kv) {
          p.kh = 0;
          p.span = seq_span(a, ++p.b);
        }
      }
    } while ((p.tiles = Shape::tiles(a, p.span, p.mb)) == 0);
  }
  __device__ static int first_of(int c, int total, int ctas) { return (int)((int64_t)c * total / ctas); }
  __device__ static int cta_of(int t, int total, int ctas) { return (int)((((int64_t)t + 1) * ctas - 1) / total); }
};

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float log2_approx(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Output row r (token r / group, head r % group) of a unit, values d, d + 1, times the gate's sigmoid.
__device__ __forceinline__ float2 load_gate2(const AttnArgs& a, int b, int kh, int r, int d) {
  const float* g = a.gate + b * a.gb + r / a.group * a.gn + (kh * a.group + r % a.group) * a.gh + d;
  return make_float2(g[0], g[1]);
}
__device__ __forceinline__ float sigmoid(float x) { return 1.f / (1.f + __expf(-x)); }
template <typename T>
__device__ __forceinline__ void store_row2(const AttnArgs& a, int b, int kh, int r, int d, float x, float y) {
  const int i = r / a.group, h = kh * a.group + r % a.group;
  T* o = static_cast<T*>(a.out) + (((int64_t)b * a.n + i) * a.heads + h) * a.dim + d;
  if constexpr (std::is_same<T, __half>::value) *reinterpret_cast<__half2*>(o) = __floats2half2_rn(x, y);
  else *reinterpret_cast<__nv_bfloat162*>(o) = __floats2bfloat162_rn(x, y);
}

// Eight values from d on.
template <typename T>
__device__ __forceinline__ void store_row8(const AttnArgs& a, int b, int kh, int r, int d, float (&f)[8]) {
  const int i = r / a.group, h = kh * a.group + r % a.group;
  if (a.gate) {
    const float* g = a.gate + b * a.gb + i * a.gn + h * a.gh + d;
    float w[8];
    if (reinterpret_cast<uintptr_t>(g) % 16 == 0) {
      const float4 x = *reinterpret_cast<const float4*>(g), y = *reinterpret_cast<const float4*>(g + 4);
      w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w, w[4] = y.x, w[5] = y.y, w[6] = y.z, w[7] = y.w;
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) w[e] = g[e];
    }
#pragma unroll
    for (int e = 0; e < 8; e++) f[e] /= 1.f + __expf(-w[e]);
  }
  uint4 v;
  uint32_t* u = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
  for (int e = 0; e < 4; e++) {
    if constexpr (std::is_same<T, __half>::value) {
      const __half2 h2 = __floats2half2_rn(f[2 * e], f[2 * e + 1]);
      u[e] = *reinterpret_cast<const uint32_t*>(&h2);
    } else {
      const __nv_bfloat162 h2 = __floats2bfloat162_rn(f[2 * e], f[2 * e + 1]);
      u[e] = *reinterpret_cast<const uint32_t*>(&h2);
    }
  }
  *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + (((int64_t)b * a.n + i) * a.heads + h) * a.dim + d) = v;
}

}  // namespace gsq
