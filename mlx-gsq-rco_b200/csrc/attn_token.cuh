// Attention over the quantised cache for few rows per key/value head (n *
// group <= 16: single tokens, small trees; more as several units of 16).
//
// Bound: HBM bytes of the cache, each read once.  At 6.5 TB/s an SM receives
// about 23 codes a cycle, so what is done per code has to stay small:
//   - codes go to fp16 exactly (2 to 3 operations per pair) and their scales,
//     one per position, are applied to the 16 x 8 tile of scores (keys) and
//     weights (values), not to the codes;
//   - both products run on mma.m16n8k16 with the codes as the 16-row operand
//     (S^T = K Q^T, O^T = V^T P^T), so 8 query rows fill the tile that a
//     token's 1 to 8 heads need, where the query as the 16-row operand (or
//     128 rows of tcgen05) would be mostly padding;
//   - each warp runs its own softmax over its own 16 positions of a tile of
//     64, so no barrier or exchange between warps interrupts the stream; the
//     four are joined once per unit of work.
// Every warp copies its own 16 rows of K and V through a private ring
// (cp.async, positions past the end filled with zeros), with 16-byte units
// exchanged by the row so that all shared loads are 16 bytes and free of
// conflicts.
//
// Weights p are rounded to fp16 (2^-11 each) for the second product; the sum
// of weights is of the unrounded ones, in fp32.  The values' scales differ by
// position, so the rounded weight is 2^15 p vs / 2^ref with a reference per
// row that follows s + log2(vs): no weight that matters leaves fp16's normal
// range, whatever the scales.  The sum of weights is relative to 2^(ref + 36):
// where ref comes from a scale up to 2^57, the weights that count in it, 2^-32
// of the largest and more, are then 2^-126 and more; and where scores that do
// not move ref have scales down to 2^-143 (below, a value is 0 in 16 bits), at
// most 2^107 each.  Where a tile with a larger scale moves ref, the warp's sums
// have references of their own from there on, in each thread (no exchanges);
// their distance from ref is then that of two scores, which fp32 tells to 2^-7
// for scores up to 2^17.
//
// The work is divided in one of two ways.  UNITS: one cluster of 1 to 8 CTAs
// for up to 16 rows of a sequence's head, whose CTAs take a share of its
// positions each and are joined through distributed shared memory; one launch,
// no scratch.  Else the tiles of all units are split evenly over the CTAs, and
// a unit that falls into several is joined by a second launch: for long caches,
// where units of very different length would leave SMs idle.
//
// Measured: 24 sequences of up to 65536 positions, 32 heads on 4 of 128, int8
// 228 us (5.2 TB/s); one of 131071, 24 heads on 4 of 256, e4m3 57 us (4.8 TB/s,
// the join included); 64 ragged ones of up to 2304 54 us.
#pragma once

#include "attn_common.cuh"

namespace gsq {

constexpr int AT_WARPS = 4;  // of a CTA, two CTAs on an SM: one is read for while the other joins its warps
constexpr int AT_TILE = 16 * AT_WARPS;
// log2 of what the sums of weights are relative to, over what the sums of values are (but for 2^15); what brings these to
// those; the scales that this does not serve
constexpr float AT_GAP = 36.f, AT_OVER = 0x1p-51f, AT_HUGE = 0x1p57f;
constexpr float AT_LOWEST = -3.402823466e38f;  // m of a row that has seen nothing

template <int D, int NT>
struct AtGeom {
  static constexpr int ROWS = 8 * NT;
  static constexpr int STAGE = 2 * 16 * D + 2 * 16 * 4;  // K, V, scales of 16 positions
  static constexpr int CTAS = D == 128 && NT == 1 ? 3 : 2;  // on an SM (registers)
  static constexpr int STAGES = D == 256 ? 3 : NT == 1 ? 4 : 6;
  static constexpr int RING = AT_WARPS * STAGES * STAGE;
  static constexpr int STAT = AT_WARPS * ROWS * 2 * 4;
  static constexpr int QFRAG = NT == 1 ? 0 : D / 16 * 32 * 8 * NT;
  static constexpr int SMEM = RING + STAT + QFRAG + ROWS * 2 * 4;
  static_assert(STAGE >= 8 * D * 4, "a stage holds the sums of eight rows");
  static_assert(CTAS * (SMEM + 1024) <= 228 * 1024, "CTAs on an SM");
};

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// 16 (or 4) bytes global -> shared; zeros where !in (the source is not read).
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async16_zfill(uint32_t dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async4_zfill(void* dst, const void* src, bool in) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(in ? 4 : 0) : "memory");
}
// 16-byte unit u of position p within a warp's 16 rows: rows p and p + 1 differ in bit 2 (the keys' loads read units
// 4c .. 4c + 3 of two neighbouring rows at a time), rows p, p + 2, p + 4, p + 6 in bits 1 and 2 (the values' loads
// read two units of four rows).
__device__ __forceinline__ int at_unit(int p, int u) { return u ^ ((p & 6) ^ (p & 1) << 2); }

struct AtShape {  // all rows of a head together
  static constexpr int ROWS = 16;
  __device__ static int blocks(const AttnArgs&) { return 1; }
  __device__ static int tiles(const AttnArgs&, const SeqSpan& s, int) { return (int)((s.len + AT_TILE - 1) / AT_TILE); }
};
using AtList = TileList<AtShape>;

// One row's eight values of q from dimension d on; zeros for rows that are not there.
template <typename T>
__device__ __forceinline__ uint4 load_q8(const AttnArgs& a, int b, int kh, int r, int d) {
  if (r >= a.n * a.group) return make_uint4(0u, 0u, 0u, 0u);
  return *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + b * a.qb + (r / a.group) * a.qn +
                                         (kh * a.group + r % a.group) * a.qh + d);
}
template <typename T>
__device__ __forceinline__ void q8_values(const uint4& v, float* f) {
  const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
  for (int i = 0; i < 8; i++) f[i] = to_f32(e[i]);
}

// bf16 queries are held in fp16 times a power of two that brings the row's largest value to [2^13, 2^14): exact but
// for values 2^27 times smaller than the largest.  Returns that power's exponent.
__device__ __forceinline__ int q_shift(float amax) {
  const int e = (int)(__float_as_uint(amax) >> 23 & 255);
  return e == 0 || e == 255 ? 0 : min(13 - (e - 127), 126);
}
__device__ __forceinline__ float exp2_int(int e) { return __int_as_float((e + 127) << 23); }  // -126 .. 127

// x 2^d, d <= 0, where 2^d may be below fp32's range and the product not.
__device__ __forceinline__ float shrunk(float x, float d) {
  const float r = exp2_approx(0.5f * d);
  return x * r * r;
}
// Adds the weights of two scores to (at, sum).
__device__ __forceinline__ void add_weights(float& at, float& sum, float s0, float s1) {
  const float next = fmaxf(at, fmaxf(s0, s1));
  sum = shrunk(sum, at - next) + exp2_approx(s0 - next) + exp2_approx(s1 - next);
  at = next;
}
// Adds another part's (reference, sum) to (top, sum). No position seen: reference -inf, sum 0 (or NaN).
__device__ __forceinline__ void add_stat(float& top, float& sum, float t2, float s2) {
  const float next = fmaxf(top, t2);
  sum = (top == next || top == -INFINITY ? sum : shrunk(sum, top - next)) +
        (t2 == next || t2 == -INFINITY ? s2 : shrunk(s2, t2 - next));
  top = next;
}
// What a part's sums are multiplied with: to the common reference, 1 where it has seen nothing (its sums are 0, or NaN).
__device__ __forceinline__ float part_factor(float m, float top) { return m == -INFINITY ? 1.f : exp2_approx(m - top); }

// Zeros for rows r0 .. r1 of a unit.
template <typename T, int D>
__device__ __forceinline__ void zero_unit(const AttnArgs& a, int b, int kh, int r0, int r1) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int r = r0 + warp; r < r1; r += blockDim.x / 32)
    for (int d = 2 * lane; d < D; d += 64) store_row2<T>(a, b, kh, r, d, 0.f, 0.f);
}

__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Two floats at the address that p has in this CTA, of CTA `rank` of the cluster.
__device__ __forceinline__ float2 ld_cluster2(const float* p, int rank) {
  uint32_t remote;
  float2 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(remote) : "memory");
  return v;
}

template <typename T, int FMT, int D, int NT, bool UNITS>
__global__ void __launch_bounds__(32 * AT_WARPS, AtGeom<D, NT>::CTAS) attn_token_kernel(const AttnArgs a) {
  using G = AtGeom<D, NT>;
  constexpr int CH = D / 64;   // 64-dimension chunks of the first product
  constexpr int MT = D / 16;   // 16-dimension tiles of the second
  extern __shared__ __align__(128) uint8_t smem[];
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint8_t* ring = smem + warp * G::STAGES * G::STAGE;
  float* stat = reinterpret_cast<float*>(smem + G::RING);  // [warp][row][m, l]
  uint2* qfrag = reinterpret_cast<uint2*>(smem + G::RING + G::STAT);

  int first, last, r0 = 0, rows = a.n * a.group;  // rows of the unit, from r0 on
  Place get = {};
  if constexpr (UNITS) {
    const int unit = blockIdx.x / a.cluster, rank = blockIdx.x % a.cluster;  // rank == %cluster_ctarank
    get.b = unit / (a.kv * a.blocks);
    get.kh = unit / a.blocks % a.kv;
    r0 = unit % a.blocks * G::ROWS;
    rows = min(rows - r0, G::ROWS);
    get.span = seq_span(a, get.b);
    get.tiles = AtShape::tiles(a, get.span, 0);
    if (get.tiles == 0) {  // the whole cluster
      if (rank == 0) zero_unit<T, D>(a, get.b, get.kh, r0, r0 + rows);
      return;
    }
    get.tile = first = rank * get.tiles / a.cluster;
    last = (rank + 1) * get.tiles / a.cluster;
  } else {
    const int total = AtList::total(a), ctas = min(a.ctas, total);
    if ((int)blockIdx.x >= ctas) {
      if (threadIdx.x == 0) a.joints[blockIdx.x].parts = 0;
      return;
    }
    first = AtList::first_of(blockIdx.x, total, ctas);
    last = AtList::first_of(blockIdx.x + 1, total, ctas);
    get = AtList::locate(a, first);
    if (threadIdx.x == 0) AtList::note(a, blockIdx.x, first, get, total, ctas);
  }
  Place use = get;

  // A warp's 16 positions of K and V, copied STEP rows at a time, a 16-byte unit a lane.
  constexpr int U = D / 16, STEP = 32 / U;
  const uint32_t lane_dst = smem_u32(ring) + lane / U * D + at_unit(lane / U, lane % U) * 16;
  int fetched = first, put = 0;
  auto fetch = [&]() {
    if (fetched < last) {
      const uint32_t st = put * G::STAGE;
      const int p0 = get.tile * AT_TILE + warp * 16, left = get.span.len - p0;  // positions of this warp that exist
      const int64_t row0 = ((int64_t)get.b * a.kv + get.kh) * a.cap + p0;
      const uint8_t *kp = a.kc + row0 * D + lane * 16, *vp = a.vc + row0 * D + lane * 16;
      if (left >= 16) {
#pragma unroll
        for (int i = 0; i < 16 / STEP; i++) {
          const uint32_t dst = (lane_dst ^ (i * STEP & 6) << 4) + st + i * STEP * D;
          cp_async16(dst, kp + i * STEP * D);
          cp_async16(dst + 16 * D, vp + i * STEP * D);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 16 / STEP; i++) {
          const uint32_t dst = (lane_dst ^ (i * STEP & 6) << 4) + st + i * STEP * D;
          const bool in = i * STEP + lane / U < left;
          cp_async16_zfill(dst, in ? kp + i * STEP * D : a.kc, in);
          cp_async16_zfill(dst + 16 * D, in ? vp + i * STEP * D : a.vc, in);
        }
      }
      const bool in = (lane & 15) < left;
      cp_async4_zfill(ring + st + 32 * D + lane * 4, (lane < 16 ? a.ks : a.vs) + (in ? row0 + (lane & 15) : 0), in);
      if (++get.tile == get.tiles && fetched + 1 < last && !UNITS) AtList::next_unit(a, get);
    }
    fetched++;
    put = put + 1 == G::STAGES ? 0 : put + 1;
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < G::STAGES - 1; i++) fetch();
  int coming = 0, read = 0;  // the stage that is read next, and the one read last, free until the next copy

  uint32_t qr[NT == 1 ? MT : 1][2];
  float factor[NT][2];  // of the scores of rows 8x + 2t, 8x + 2t + 1, to base 2
  int lim[NT][2];       // tree: prefix ends; causal: positions the row sees (relative to the prefix end)
  float o[MT][NT][4], m[NT][2], l[NT][2];  // o relative to 2^(m - AT_GAP - 15), l to 2^m
  float at[NT][2], own[NT][2];  // a thread's own reference and sum of weights
  uint4 raw[NT][2 * CH];  // q of the coming unit: row 8x + g, dimensions 64c + 16t ..
  auto fetch_q = [&]() {
#pragma unroll
    for (int x = 0; x < NT; x++)
#pragma unroll
      for (int c = 0; c < 2 * CH; c++)
        raw[x][c] = load_q8<T>(a, use.b, use.kh, r0 + 8 * x + g, 64 * (c / 2) + 16 * t + 8 * (c % 2));
  };
  fetch_q();

  for (int tile = first; tile < last || UNITS;) {
    // ---- a unit's run of tiles ----
    const int b = use.b, kh = use.kh;
    const SeqSpan span = use.span;
    const bool whole = UNITS ? a.cluster == 1 : use.tile == 0 && tile + use.tiles <= last;
    const int slot = 2 * blockIdx.x + (tile == first ? 0 : 1);
    const int end = min(last, tile + use.tiles - use.tile);
    bool wide = false;  // m may come from a scale above AT_HUGE: at and own instead of m and l
#pragma unroll
    for (int x = 0; x < NT; x++) {
      float amax = 0.f;
      float qv[CH][16];
#pragma unroll
      for (int c = 0; c < CH; c++) {
        q8_values<T>(raw[x][2 * c], qv[c]);
        q8_values<T>(raw[x][2 * c + 1], qv[c] + 8);
#pragma unroll
        for (int e = 0; e < 16; e++) amax = fmaxf(amax, fabsf(qv[c][e]));
      }
      int shift = 0;
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        shift = q_shift(amax);
        const float up = exp2_int(shift);
#pragma unroll
        for (int c = 0; c < CH; c++)
#pragma unroll
          for (int e = 0; e < 16; e++) qv[c][e] *= up;
      }
#pragma unroll
      for (int c = 0; c < CH; c++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const __half2 h0 = __floats2half2_rn(qv[c][4 * j], qv[c][4 * j + 1]);
          const __half2 h1 = __floats2half2_rn(qv[c][4 * j + 2], qv[c][4 * j + 3]);
          const uint32_t b0 = *reinterpret_cast<const uint32_t*>(&h0), b1 = *reinterpret_cast<const uint32_t*>(&h1);
          if constexpr (NT == 1) {
            qr[4 * c + j][0] = b0;
            qr[4 * c + j][1] = b1;
          } else if (warp == x) {
            qfrag[((4 * c + j) * NT + x) * 32 + lane] = make_uint2(b0, b1);
          }
        }
#pragma unroll
      for (int c = 0; c < 2; c++) {
        const int r = 8 * x + 2 * t + c;  // this lane's columns of the score tile; their shift is held by lanes 4r'
        factor[x][c] = a.scale * 1.4426950408889634f * exp2_int(-__shfl_sync(0xffffffffu, shift, 4 * (2 * t + c)));
        lim[x][c] = (r0 + r) / a.group;
        m[x][c] = AT_LOWEST;
        l[x][c] = 0.f;
      }
    }
    if constexpr (NT > 1) __syncthreads();
#pragma unroll
    for (int j = 0; j < MT; j++)
#pragma unroll
      for (int x = 0; x < NT; x++)
#pragma unroll
        for (int e = 0; e < 4; e++) o[j][x][e] = 0.f;

    for (; tile < end; tile++) {
      __syncwarp();  // every lane has read the stage that is filled next
      fetch();
      cp_async_wait<G::STAGES - 1>();
      __syncwarp();
      const uint8_t* st = ring + coming * G::STAGE;
      read = coming;
      coming = coming + 1 == G::STAGES ? 0 : coming + 1;
      const int p0 = use.tile * AT_TILE + warp * 16;
      use.tile++;
      if (p0 >= span.len) continue;
      const float* sc = reinterpret_cast<const float*>(st + 32 * D);

      float s[NT][4], s2[NT][4];  // two chains of products
#pragma unroll
      for (int x = 0; x < NT; x++)
#pragma unroll
        for (int e = 0; e < 4; e++) s[x][e] = s2[x][e] = 0.f;
#pragma unroll
      for (int c = 0; c < CH; c++) {
        const uint4 ka = *reinterpret_cast<const uint4*>(st + g * D + at_unit(g, 4 * c + t) * 16);
        const uint4 kb = *reinterpret_cast<const uint4*>(st + (g + 8) * D + at_unit(g + 8, 4 * c + t) * 16);
        const uint32_t* wa = reinterpret_cast<const uint32_t*>(&ka);
        const uint32_t* wb = reinterpret_cast<const uint32_t*>(&kb);
#pragma unroll
        for (int j = 0; j < 4; j++) {
          uint32_t a0, a1, a2, a3;
          codes_to_half2<FMT>(wa[j], a0, a2);
          codes_to_half2<FMT>(wb[j], a1, a3);
#pragma unroll
          for (int x = 0; x < NT; x++) {
            if constexpr (NT == 1) {
              mma_f16(j & 1 ? s2[x] : s[x], a0, a1, a2, a3, qr[4 * c + j][0], qr[4 * c + j][1]);
            } else {
              const uint2 q2 = qfrag[((4 * c + j) * NT + x) * 32 + lane];
              mma_f16(j & 1 ? s2[x] : s[x], a0, a1, a2, a3, q2.x, q2.y);
            }
          }
        }
      }
      // scores to base 2; s[x][e]: position p0 + g + 8 (e / 2), row 8x + 2t + e % 2
      const float ks0 = sc[g], ks1 = sc[g + 8];
      // (of scale 0, whose vector has a part in the sum of weights only, as 2^-100, so that that sum stays finite, and with
      // no weight in the other, whatever its codes)
      const float lv0 = log2_approx(sc[16 + g] > 0.f ? sc[16 + g] : 0x1p-100f);
      const float lv1 = log2_approx(sc[24 + g] > 0.f ? sc[24 + g] : 0x1p-100f);
      const float nan0 = sc[16 + g] - sc[16 + g], nan1 = sc[24 + g] - sc[24 + g];  // NaN where the scale is
      const float lr0 = lv0 + AT_GAP, lift0 = (sc[16 + g] > 0.f ? 15.f : -INFINITY) + nan0;
      const float lr1 = lv1 + AT_GAP, lift1 = (sc[24 + g] > 0.f ? 15.f : -INFINITY) + nan1;
      const bool edge = p0 + 16 > span.base || p0 + 16 > span.len;  // warp-uniform: some row may not see all of these
      uint32_t pb[NT][2];
#pragma unroll
      for (int x = 0; x < NT; x++) {
#pragma unroll
        for (int e = 0; e < 4; e++) s[x][e] = (s[x][e] + s2[x][e]) * ((e < 2 ? ks0 : ks1) * factor[x][e & 1]);
        if (edge) {
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const int p = p0 + g + (e < 2 ? 0 : 8);
            const int off = p - span.base;  // index among the new tokens
            bool see = p < span.len;
            if (off >= 0 && see) {
              const int i = lim[x][e & 1];
              see = i < span.count;
              if (!a.tree) see = see && off <= i;
              else if (see)
                see = (uint32_t)a.tree[b * a.tree_stride + (int64_t)i * a.words + (off >> 5)] >> (off & 31) & 1;
            }
            if (!see) s[x][e] = -INFINITY;
          }
        }
        // the row's reference: the largest of u = s + log2(vs) + AT_GAP (itself, so that the largest weight, 2^15, needs no
        // rounding to fp16: rounded up to a whole number it moves less often, but the error of the outputs grows by a third).
        // Both weights come from u - m, so that they fit each other where s is so large that u has lost what was added.
        float lo[2], u[4];
#pragma unroll
        for (int e = 0; e < 4; e++) u[e] = s[x][e] + (e < 2 ? lr0 : lr1);
#pragma unroll
        for (int c = 0; c < 2; c++) {
          float r = fmaxf(fmaxf(u[c], u[2 + c]), m[x][c]);
          r = fmaxf(r, __shfl_xor_sync(0xffffffffu, r, 4));
          r = fmaxf(r, __shfl_xor_sync(0xffffffffu, r, 8));
          r = fmaxf(r, __shfl_xor_sync(0xffffffffu, r, 16));
          lo[c] = r;
        }
        const bool grew = lo[0] > m[x][0] || lo[1] > m[x][1] || wide;
        if (__any_sync(0xffffffffu, grew)) {
          if (!wide && __any_sync(0xffffffffu, fmaxf(sc[16 + g], sc[24 + g]) > AT_HUGE)) {
            wide = true;
#pragma unroll
            for (int y = 0; y < NT; y++)
#pragma unroll
              for (int c = 0; c < 2; c++) {
                // (brought to 1 .. 2: beside m it may be 2^-100 times smaller)
                const int power = min((int)(__float_as_uint(l[y][c]) >> 23 & 255), 253) - 127;
                const bool some = l[y][c] > 0.f;
                at[y][c] = some ? m[y][c] + (float)max(power, -126) : AT_LOWEST;
                own[y][c] = some ? l[y][c] * exp2_int(-max(power, -126)) : l[y][c];
              }
          }
          if (wide) {
#pragma unroll
            for (int c = 0; c < 2; c++) add_weights(at[x][c], own[x][c], s[x][c], s[x][2 + c]);
          }
          const float r0 = exp2_approx(0.5f * (m[x][0] - lo[0])), f0 = r0 * r0;
          const float r1 = exp2_approx(0.5f * (m[x][1] - lo[1])), f1 = r1 * r1;
          l[x][0] = l[x][0] * r0 * r0;  // (f0 may be below fp32's range where this is not)
          l[x][1] = l[x][1] * r1 * r1;
          m[x][0] = lo[0];
          m[x][1] = lo[1];
#pragma unroll
          for (int j = 0; j < MT; j++) {
            o[j][x][0] *= f0;
            o[j][x][1] *= f1;
            o[j][x][2] *= f0;
            o[j][x][3] *= f1;
          }
        }
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const float d = u[e] - m[x][e & 1];  // -inf where hidden
          l[x][e & 1] += exp2_approx(d - (e < 2 ? lr0 : lr1));
          w[e] = s[x][e] == -INFINITY ? 0.f : exp2_approx(d + (e < 2 ? lift0 : lift1));
        }
        const __half2 h0 = __floats2half2_rn(w[0], w[1]), h1 = __floats2half2_rn(w[2], w[3]);
        pb[x][0] = transpose8x8(*reinterpret_cast<const uint32_t*>(&h0));
        pb[x][1] = transpose8x8(*reinterpret_cast<const uint32_t*>(&h1));
      }
      // O^T += V^T P^T: rows of tile 8h + j are dimensions 128h + 16g + 2j (registers 0, 1) and + 1 (2, 3)
#pragma unroll
      for (int h = 0; h < D / 128; h++) {
        uint4 v[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int p = 2 * t + (i & 1) + (i >> 1) * 8;
          v[i] = *reinterpret_cast<const uint4*>(st + 16 * D + p * D + at_unit(p, 8 * h + g) * 16);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const uint32_t w0 = reinterpret_cast<const uint32_t*>(&v[0])[i], w1 = reinterpret_cast<const uint32_t*>(&v[1])[i];
          const uint32_t w2 = reinterpret_cast<const uint32_t*>(&v[2])[i], w3 = reinterpret_cast<const uint32_t*>(&v[3])[i];
          uint32_t a0, a1, a2, a3;
          codes_to_half2<FMT>(__byte_perm(w0, w1, 0x5140), a0, a1);
          codes_to_half2<FMT>(__byte_perm(w2, w3, 0x5140), a2, a3);
#pragma unroll
          for (int x = 0; x < NT; x++) mma_f16(o[8 * h + 2 * i][x], a0, a1, a2, a3, pb[x][0], pb[x][1]);
          codes_to_half2<FMT>(__byte_perm(w0, w1, 0x7362), a0, a1);
          codes_to_half2<FMT>(__byte_perm(w2, w3, 0x7362), a2, a3);
#pragma unroll
          for (int x = 0; x < NT; x++) mma_f16(o[8 * h + 2 * i + 1][x], a0, a1, a2, a3, pb[x][0], pb[x][1]);
        }
      }
    }

    // ---- join the warps. Each puts its sums into the stage it has just read, in the fragments' order with the lanes
    // exchanged by the tile, and warp w adds all warps' up for dimensions 16w .. and 64 + 16w .. of every 128: lane
    // (jj, tt) for dimensions 2jj, 2jj + 1 of rows 2tt, 2tt + 1, free of conflicts on both sides.
    constexpr int PIECES = D / (16 * AT_WARPS);
    const int tt = lane & 3, jj = lane >> 2;
    float2 gate[NT][2][PIECES];
    if (whole && a.gate) {
#pragma unroll
      for (int x = 0; x < NT; x++)
#pragma unroll
        for (int c = 0; c < 2; c++)
#pragma unroll
          for (int i = 0; i < PIECES; i++) {
            const int r = 8 * x + 2 * tt + c;
            gate[x][c][i] =
                r < rows ? load_gate2(a, b, kh, r0 + r, 16 * (warp + i * AT_WARPS) + 2 * jj) : make_float2(0.f, 0.f);
          }
    }
#pragma unroll
    for (int x = 0; x < NT; x++)
#pragma unroll
      for (int c = 0; c < 2; c++) {
        if (wide) {
          // both sums relative to 2^row, the largest of the lanes' references, or where values are large to 2^(row + 80):
          // fp32 has a place for them there
          float row = at[x][c];
#pragma unroll
          for (int i = 4; i < 32; i <<= 1) row = fmaxf(row, __shfl_xor_sync(0xffffffffu, row, i));
          const bool large = m[x][c] > row;
          l[x][c] = shrunk(own[x][c], at[x][c] - row) * (large ? 0x1p-80f : 1.f);
          row += large ? 80.f : 0.f;
          const float r = exp2_approx(0.5f * (m[x][c] - row));  // (1 where both are AT_LOWEST, and o is 0)
#pragma unroll
          for (int j = 0; j < MT; j++) {
            o[j][x][c] = o[j][x][c] * r * r;
            o[j][x][c + 2] = o[j][x][c + 2] * r * r;
          }
          if (m[x][c] != AT_LOWEST) m[x][c] = row;
        }
        if (m[x][c] == AT_LOWEST) m[x][c] = -INFINITY;
#pragma unroll
        for (int i = 4; i < 32; i <<= 1) l[x][c] += __shfl_xor_sync(0xffffffffu, l[x][c], i);
        if (g == 0)
          *reinterpret_cast<float2*>(stat + (warp * G::ROWS + 8 * x + 2 * t + c) * 2) = make_float2(m[x][c], l[x][c]);
      }
    __syncthreads();
    const int spare = UNITS ? 0 : read * G::STAGE;  // (UNITS: every stage is free at the end)
    // UNITS: the CTA's sums of rows 8x .., in the last stage of warp x, the same place in every CTA
    auto result = [&](int x) {
      return reinterpret_cast<float*>(smem + x * G::STAGES * G::STAGE + (G::STAGES - 1) * G::STAGE);
    };
    float* unit_stat = reinterpret_cast<float*>(smem + G::RING + G::STAT + G::QFRAG);
    float* mine = reinterpret_cast<float*>(ring + spare);
    const float* all = reinterpret_cast<const float*>(smem + spare);  // warp w's is w * STAGES * STAGE bytes on
    if (!UNITS && tile < last) AtList::next_unit(a, use);
#pragma unroll
    for (int x = 0; x < NT; x++) {
      if (x > 0) __syncthreads();  // the stages have been read
#pragma unroll
      for (int c = 0; c < 2; c++) {
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < AT_WARPS; w++) top = fmaxf(top, stat[(w * G::ROWS + 8 * x + 2 * t + c) * 2]);
        const float f = m[x][c] == -INFINITY ? 1.f : exp2_approx(m[x][c] - top);  // no weight: 0, or NaN
#pragma unroll
        for (int j = 0; j < MT; j++) {
          mine[(j * 4 + c) * 32 + (lane ^ (j & 7) << 2)] = o[j][x][c] * f;
          mine[(j * 4 + c + 2) * 32 + (lane ^ (j & 7) << 2)] = o[j][x][c + 2] * f;
        }
      }
      if (!UNITS && x == NT - 1 && tile < last) fetch_q();  // of the next unit, while this one is joined
      __syncthreads();
#pragma unroll
      for (int c = 0; c < 2; c++) {
        const int r = 8 * x + 2 * tt + c;
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < AT_WARPS; w++) top = fmaxf(top, stat[(w * G::ROWS + r) * 2]);
#pragma unroll
        for (int w = 0; w < AT_WARPS; w++) {
          const float2 s = *reinterpret_cast<const float2*>(stat + (w * G::ROWS + r) * 2);
          sum += s.x == -INFINITY ? s.y : shrunk(s.y, s.x - top);
        }
        const bool none = sum == 0.f || (r0 + r) / a.group >= span.count;
        const float inv = none ? 0.f : 1.f / sum;
#pragma unroll
        for (int i = 0; i < PIECES; i++) {
          const int piece = warp + i * AT_WARPS, h = piece / 8;  // dimensions 16 piece ..
          const float* p = all + ((8 * h + jj) * 4 + c) * 32 + (((piece & 7) ^ jj) << 2 | tt);
          float v0 = 0.f, v1 = 0.f;
#pragma unroll
          for (int w = 0; w < AT_WARPS; w++) {
            v0 += p[w * (G::STAGES * G::STAGE / 4)];
            v1 += p[w * (G::STAGES * G::STAGE / 4) + 64];
          }
          const int d = 16 * piece + 2 * jj;
          if (r >= rows) continue;
          if (whole) {
            const float f0 = a.gate ? inv * sigmoid(gate[x][c][i].x) : inv;
            const float f1 = a.gate ? inv * sigmoid(gate[x][c][i].y) : inv;
            store_row2<T>(a, b, kh, r0 + r, d, none ? 0.f : v0 * AT_OVER * f0, none ? 0.f : v1 * AT_OVER * f1);
          } else if constexpr (UNITS) {
            *reinterpret_cast<float2*>(result(x) + (2 * tt + c) * D + d) = make_float2(v0, v1);
            if (piece == 0 && jj == 0) *reinterpret_cast<float2*>(unit_stat + r * 2) = make_float2(top, sum);
          } else {
            *reinterpret_cast<float2*>(a.part + ((int64_t)slot * G::ROWS + r) * D + d) =
                make_float2(v0 * AT_OVER, v1 * AT_OVER);
            if (piece == 0 && jj == 0)
              *reinterpret_cast<float2*>(a.stat + ((int64_t)slot * G::ROWS + r) * 2) = make_float2(top, sum);
          }
        }
      }
    }
    if constexpr (UNITS) {
      if (whole) return;
      // every CTA of the cluster takes its share of the outputs from all of them
      cluster_sync_all();
      const int ctas = a.cluster, rank = blockIdx.x % ctas;
      for (int i = rank * 32 * AT_WARPS + threadIdx.x; i < rows * (D / 2); i += ctas * 32 * AT_WARPS) {
        const int r = i / (D / 2), d = i % (D / 2) * 2;
        float2 s[8], v[8];
#pragma unroll
        for (int k = 0; k < 8; k++) {
          if (k >= ctas) continue;
          s[k] = ld_cluster2(unit_stat + r * 2, k);
          v[k] = ld_cluster2(result(r / 8) + r % 8 * D + d, k);
        }
        float2 gate2 = a.gate ? load_gate2(a, b, kh, r0 + r, d) : make_float2(0.f, 0.f);
        float top = -INFINITY, sum = 0.f, x = 0.f, y = 0.f;
#pragma unroll
        for (int k = 0; k < 8; k++)
          if (k < ctas) add_stat(top, sum, s[k].x, s[k].y);
#pragma unroll
        for (int k = 0; k < 8; k++) {
          if (k >= ctas) continue;
          const float f = part_factor(s[k].x, top);
          x = fmaf(v[k].x, f, x);
          y = fmaf(v[k].y, f, y);
        }
        const bool none = sum == 0.f || (r0 + r) / a.group >= span.count;
        const float inv = none ? 0.f : 1.f / sum;
        const float f0 = a.gate ? inv * sigmoid(gate2.x) : inv, f1 = a.gate ? inv * sigmoid(gate2.y) : inv;
        store_row2<T>(a, b, kh, r0 + r, d, none ? 0.f : x * AT_OVER * f0, none ? 0.f : y * AT_OVER * f1);
      }
      cluster_sync_all();  // no CTA leaves while another may read its shared memory
      return;
    }
    __syncthreads();  // the stages and stat are free
  }
}

// Joins the partial results of the units that fell into several CTAs, in CTA order, and writes zeros for the rows
// that no tile reaches. CTAs (c, 0 ..): the unit that CTA c noted. 1 to 8 of their warps take a row together, each some
// of its parts, D / 32 values a lane: as many as there are for the rows, since what bounds this is the chain of loads
// along the parts.
template <typename T, int D, typename Shape>
__global__ void __launch_bounds__(256) attn_join_kernel(const AttnArgs a) {
  constexpr int NV = D / 32;
  __shared__ float acc[8][D];
  pdl_launch_dependents();
  pdl_wait();
  const int rows = a.n * a.group, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (blockIdx.y == 0) {
    const int blocks = Shape::blocks(a);
    for (int i = blockIdx.x; i < a.batch * blocks; i += gridDim.x) {
      const int b = i / blocks, mb = i % blocks;
      if (Shape::tiles(a, seq_span(a, b), mb) == 0)
        for (int kh = 0; kh < a.kv; kh++) zero_unit<T, D>(a, b, kh, mb * Shape::ROWS, min(rows, (mb + 1) * Shape::ROWS));
    }
  }
  const Joint j = a.joints[blockIdx.x];
  if (j.parts == 0) return;
  const int r0 = j.mb * Shape::ROWS, count = min(rows - r0, Shape::ROWS), warps = 8 * gridDim.y;
  int share = 1;
  while (share < 8 && 2 * share * count <= warps && 4 * share <= j.parts) share *= 2;
  for (int base = 0; base < count; base += warps / share) {  // the same for the whole CTA
    const int r = base + (blockIdx.y * 8 + warp) / share;
    const bool live = r < count;
    float top = -INFINITY, sum = 0.f;
    float o[NV] = {};
    if (live) {
      for (int i = lane; i < j.parts; i += 32) {
        const float2 s = *reinterpret_cast<const float2*>(a.stat + ((int64_t)j.slot(i) * a.rows8 + r) * 2);
        add_stat(top, sum, s.x, s.y);
      }
#pragma unroll
      for (int x = 16; x; x >>= 1)
        add_stat(top, sum, __shfl_xor_sync(0xffffffffu, top, x), __shfl_xor_sync(0xffffffffu, sum, x));
#pragma unroll 8
      for (int i = warp % share; i < j.parts; i += share) {
        const int64_t at = (int64_t)j.slot(i) * a.rows8 + r;
        const float f = part_factor(a.stat[at * 2], top);
#pragma unroll
        for (int e = 0; e < NV; e += 4) {
          const float4 v = *reinterpret_cast<const float4*>(a.part + at * D + lane * NV + e);
          o[e] = fmaf(v.x, f, o[e]);
          o[e + 1] = fmaf(v.y, f, o[e + 1]);
          o[e + 2] = fmaf(v.z, f, o[e + 2]);
          o[e + 3] = fmaf(v.w, f, o[e + 3]);
        }
      }
    }
    if (share > 1) {
#pragma unroll
      for (int e = 0; e < NV; e += 4)
        *reinterpret_cast<float4*>(&acc[warp][lane * NV + e]) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
      __syncthreads();
      if (warp % share == 0) {
        for (int w = 1; w < share; w++)
#pragma unroll
          for (int e = 0; e < NV; e++) o[e] += acc[warp + w][lane * NV + e];
      }
      __syncthreads();
    }
    if (!live || warp % share) continue;
    const bool none = sum == 0.f || (r0 + r) / a.group >= j.count;
    const float inv = none ? 0.f : 1.f / sum;
#pragma unroll
    for (int e = 0; e < NV; e += 2) {
      float2 f = make_float2(inv, inv);
      if (a.gate) {
        const float2 x = load_gate2(a, j.b, j.kh, r0 + r, lane * NV + e);
        f = make_float2(inv * sigmoid(x.x), inv * sigmoid(x.y));
      }
      store_row2<T>(a, j.b, j.kh, r0 + r, lane * NV + e, none ? 0.f : o[e] * f.x, none ? 0.f : o[e + 1] * f.y);
    }
  }
}

}  // namespace gsq
