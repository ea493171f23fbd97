// Attention over the quantised cache for many rows per key/value head (n *
// group > 16: chunks of a prompt, drafted trees), on tcgen05.
//
// Both products of a block of 128 rows run on the tensor core with the rows
// as M: S = Q K^T (N = 64 positions) and O += P V (N = the head's width),
// accumulators in TMEM.  Bound: the tensor core where the rows fill their
// blocks (4 D operations a row and position; at D = 256 a tile of 64
// positions takes 1024 cycles), else the bytes of the cache.  Each code is
// read, made fp16 and stored to shared memory once per row block, and that
// is what competes with the tensor core:
//   - Q and P are TMEM operands, so that the tensor core reads only K and V from
//     shared memory: per tile 64 KB written and 64 KB read, 1024 cycles of
//     its 128 bytes a cycle, where Q in shared memory would add 64 KB;
//   - K and V tiles have one layout (64 x 64 blocks of 128-byte rows, 128-byte
//     swizzle): K is read as a K-major operand, V as an MN-major one, so no
//     transposition is needed;
//   - scales stay out of the codes: a position's key scale multiplies its
//     score, and its value scale enters the weight as 2^(s + log2 vs - ref),
//     with one exponential; the sum of weights takes the same value times
//     1 / vs. From a tile with a scale outside 2^-40 .. 2^40 on, where that
//     value may leave fp32's range, the run's sums come from the scores a
//     second time, with exponentials of their own (that code costs the chunk
//     below 1.3 % of its time, in registers).
// Roles (20 warps): two softmax warpgroups, one row a thread, that take the
// two halves of every tile's columns; two that dequantise; one warp issues the
// products, one thread the bulk copies of codes (a tile is one contiguous
// piece), one warp prepares the tile's scales.  S has two tiles in TMEM, and
// P takes the place of the scores it comes from, so the next tile's scores are
// there when the softmax is through with one.
// The groups pass each other the largest score of a row's half, so that both
// follow the same reference (the running maximum). Half a tile a thread keeps
// the softmax loop, which is unrolled over its scores, short enough for the
// instruction caches: with whole tiles in turn a fifth of its time went into
// instruction misses.
// Measured (777 rows of 6 heads on each of 4, after 23224 positions of 256):
// 577 us, 782 TFLOP/s, 47 % of the tensor core's measured rate; about 2300
// cycles a tile, of which the softmax warps are busy 2000 (their instructions
// depend on one another, and two of them share an issue slot with dequantising
// warps).  Before the code for far scales, with all rows seeing all positions,
// 476 us; there, products issued by one lane with values of its own took 562,
// and scales prepared by each softmax warp for itself 542.
// The reference is followed lazily: O is rescaled only when it grows by more
// than 2^8, which weights of up to 2^14 in fp16 leave room for.
// Weights are rounded to fp16 (2^-11 each); their sum is of the unrounded
// ones, in fp32.  Every wait is bounded.
#pragma once

#include "attn_token.cuh"
#include "gsq_tc.cuh"

namespace gsq {

constexpr int AR_M = 128, AR_TILE = 64, AR_HALF = AR_TILE / 2;
constexpr int AR_SCALES = 3 * AR_HALF + 4;  // floats of half a tile's scales
constexpr int AR_GROUP = 4, AR_SOFTMAX = 2 * AR_GROUP, AR_DEQUANT = 8;  // warps
constexpr int AR_THREADS = 32 * (AR_SOFTMAX + AR_DEQUANT + 4);  // of the last four: products, copies, scales

template <int D>
struct ArGeom {
  static constexpr int ITEM = AR_TILE * D * 2;  // one K or V tile in fp16
  static constexpr int STAGES = D == 256 ? 5 : 6;
  static constexpr int RAW = AR_TILE * D;       // its codes
  static constexpr int RAWS = 3;
  static constexpr int SCALES = 4 * AR_SCALES * 4;  // of two tiles
  static constexpr int STATE = 10 * AR_M * 4;    // the two groups' maxima of two tiles, their sums and what these are relative to
  static constexpr int SMEM = 1024 + STAGES * ITEM + RAWS * RAW + SCALES + STATE + 512;
  static constexpr int O = 0, Q = D, S = Q + D / 2;  // TMEM columns; S: two tiles
  static constexpr int COLS = 512;
  static_assert(S + 2 * AR_TILE <= COLS && SMEM <= 227 * 1024, "fits");
};

struct ArShape {  // blocks of 128 rows; with a causal mask an early block sees fewer positions
  static constexpr int ROWS = AR_M;
  __device__ static int blocks(const AttnArgs& a) { return (a.n * a.group + ROWS - 1) / ROWS; }
  __device__ static int tiles(const AttnArgs& a, const SeqSpan& s, int mb) {
    if (mb * ROWS / a.group >= s.count) return 0;
    int len = s.len;
    if (!a.tree) {
      const int last = min(((mb + 1) * ROWS - 1) / a.group, s.count - 1);
      len = min(max(s.base + last + 1, 0), (int)a.cap);
    }
    return (len + AR_TILE - 1) / AR_TILE;
  }
};
using ArList = TileList<ArShape>;

// A run: the part of one unit that lies in this CTA's tiles [first, last).
struct ArRun {
  int t, last, len;  // the run's first tile; the CTA's end; tiles of the run
  bool whole;        // all of the unit
  Place at;

  __device__ void settle() {
    len = min(at.tiles - at.tile, last - t);
    whole = at.tile == 0 && len == at.tiles;
  }
  __device__ void begin(const AttnArgs& a, int first, int end) {
    t = first;
    last = end;
    at = ArList::locate(a, first);
    settle();
  }
  __device__ bool next(const AttnArgs& a) {
    t += len;
    if (t >= last) return false;
    ArList::next_unit(a, at);
    settle();
    return true;
  }
};

// ---- tcgen05 with a TMEM operand, and wide TMEM loads and stores ----

__device__ __forceinline__ void tc_mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                              uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
#define GSQ_O8(x, i) "=r"(x[i]), "=r"(x[i + 1]), "=r"(x[i + 2]), "=r"(x[i + 3]), "=r"(x[i + 4]), "=r"(x[i + 5]), \
                     "=r"(x[i + 6]), "=r"(x[i + 7])
#define GSQ_I8(x, i) "r"(x[i]), "r"(x[i + 1]), "r"(x[i + 2]), "r"(x[i + 3]), "r"(x[i + 4]), "r"(x[i + 5]), \
                     "r"(x[i + 6]), "r"(x[i + 7])
// 32 columns of this thread's lane; the load is complete after tmem_wait_ld().
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : GSQ_O8(r, 0), GSQ_O8(r, 8), GSQ_O8(r, 16), GSQ_O8(r, 24)
      : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,"
      "%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::GSQ_I8(r, 0), GSQ_I8(r, 8), GSQ_I8(r, 16),
      GSQ_I8(r, 24), "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::GSQ_I8(r, 0),
      GSQ_I8(r, 8), "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Shared-memory descriptors with 128-byte swizzle, of which only the low word depends on the address (in 16-byte units):
// K-major (8 rows of 128 bytes 1024 bytes apart from the next 8), and MN-major (rows of 64 values, 8 rows of K 1024
// bytes apart from the next 8, the next 64 values of MN `lbo` bytes on).
constexpr uint32_t AR_DESC_HI = (1024 >> 4) | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint64_t ar_desc(uint32_t lo) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(AR_DESC_HI));
  return d;
}
__device__ __forceinline__ uint32_t ar_k_major(uint32_t saddr) { return (saddr >> 4) | 1u << 16; }
__device__ __forceinline__ uint32_t ar_mn_major(uint32_t saddr, uint32_t lbo) { return (saddr >> 4) | (lbo >> 4) << 16; }
// D = fp32, A = B = fp16, M = 128; B K-major or MN-major.
__host__ __device__ constexpr uint32_t ar_idesc(int n, bool b_mn) {
  return (1u << 4) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(AR_M >> 4) << 24);
}

// One lane of the warp, the same at every call.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(one));
  return one != 0;
}

// mbar_wait_bounded with the clock read every 64 tries only: a waiting warp leaves the issue slots to the others (the
// waits were a quarter of this kernel's instructions).
__device__ __forceinline__ bool ar_wait(uint64_t* bar, uint32_t parity, int* err) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  while (true) {
#pragma unroll 1
    for (int i = 0; i < 64; i++)
      if (mbar_try_wait_sleep(bar, parity, 20000u)) return true;
    if (clock64() - t0 > (1ll << 31)) {
      if (err) atomicExch(err, DEV_WAIT_TIMEOUT);
      return false;
    }
  }
}
// A bounded wait of a whole warp: all lanes go on, or none.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* err) {
  return __all_sync(0xffffffffu, ar_wait(bar, parity, err));
}

// The two warps of 32 rows meet (hardware barriers 1 .. 4, in a fraction of an mbarrier's time). It has no limit, so a
// warp that gives up still meets the other as often as that one will wait.
__device__ __forceinline__ void ar_meet(int quarter) { asm volatile("bar.sync %0, 64;" ::"r"(quarter + 1) : "memory"); }

// Which of positions p0 .. p0 + 63 token i of sequence b sees, as bits.
__device__ __forceinline__ uint64_t ar_visible(const AttnArgs& a, int b, const SeqSpan& s, int i, int p0) {
  if (i >= s.count) return 0;
  auto below = [](int k) { return k <= 0 ? 0ull : k >= 64 ? ~0ull : (1ull << k) - 1; };
  if (!a.tree) return below(min(s.base + i + 1, s.len) - p0);
  const int off = p0 - s.base;  // of bit 0 among the new tokens
  uint64_t m = below(-off);
  const int32_t* row = a.tree + b * a.tree_stride + (int64_t)i * a.words;
  const int w0 = off >> 5;  // floor
#pragma unroll
  for (int k = 0; k < 3; k++) {
    const int w = w0 + k;
    const int shift = w * 32 - off;  // -31 .. 64
    if (w < 0 || w >= a.words || shift >= 64) continue;
    const uint64_t bits = (uint32_t)row[w];
    m |= shift < 0 ? bits >> -shift : bits << shift;
  }
  return m & below(s.len - p0);
}

// Whether a value scale is outside 2^-40 .. 2^40 (0 is not). Within, one reference serves both sums: a weight relative to
// the largest of the scaled ones is within 2^80 of its size relative to the largest weight, so that those of 2^-32 and
// more, which count in the sum, are 2^-112 and more, within fp32's range.
__device__ __forceinline__ bool far_scale(float v) { return v > 0.f && (v < 0x1p-40f || v > 0x1p40f); }

// Scales of a tile's positions p and p + 32, one a lane, as the softmax uses them: the key's times a factor, log2 of the
// value's and its inverse in linear terms (not used where `wide`), and which of a half's value scales are 0 (bits).
struct ArScales {
  float key[2], log[2], inverse[2];
  uint32_t zeros[2];

  __device__ __forceinline__ void set(const float (&k)[2], const float (&v)[2], float factor, bool wide) {
#pragma unroll
    for (int h = 0; h < 2; h++) {
      // A vector of scale 0 has no part in the output, but in the sum of weights: where that is taken from the scaled
      // weights it is weighted with the smallest scale beside it (a larger one would move the
      // reference of rows that do not see its vector), and that weight left out of P. NaN stays, with 1 / vs as
      // 0, so that a row that does not see the position takes no harm.
      float lv = v[h] > 0.f ? log2_approx(v[h]) : -INFINITY;
      zeros[h] = __ballot_sync(0xffffffffu, v[h] == 0.f);
      if (zeros[h] && !wide) {
        float low = v[h] > 0.f ? lv : INFINITY;
#pragma unroll
        for (int o = 16; o; o >>= 1) low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
        if (v[h] == 0.f) lv = low == INFINITY ? -40.f : low;
      }
      const bool nan = isnan(v[h]);
      key[h] = k[h] * factor;
      log[h] = nan ? v[h] : lv;
      inverse[h] = nan ? 0.f : exp2_approx(-lv);
    }
  }
  // For each half 96 floats, its zeros and the flag.
  __device__ __forceinline__ void store(float* out, bool wide) const {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int h = 0; h < 2; h++) {
      float* to = out + h * AR_SCALES;
      to[lane] = key[h];
      to[AR_HALF + lane] = log[h];
      to[2 * AR_HALF + lane] = inverse[h];
      if (lane == 0) *reinterpret_cast<uint2*>(to + 3 * AR_HALF) = make_uint2(zeros[h], wide);
    }
  }
};

template <typename T, int FMT, int D>
__global__ void __launch_bounds__(AR_THREADS, 1) attn_rows_kernel(const AttnArgs a) {
  using G = ArGeom<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);  // (an offset: the pointer stays a shared one)
  uint8_t* raw = smem + G::STAGES * G::ITEM;
  float* scales = reinterpret_cast<float*>(raw + G::RAWS * G::RAW);  // [tile & 1][half][ks | log2 vs | 1 / vs | zeros, wide]
  float* tops = scales + G::SCALES / 4;   // [tile & 1][group][128]: largest scores, to base 2
  float* sums = tops + 4 * AR_M;          // [group][128]
  float2* mores = reinterpret_cast<float2*>(sums + 2 * AR_M);  // [group][128]: the sum is relative to 2^(x + y)
  uint64_t* bars = reinterpret_cast<uint64_t*>(mores + 2 * AR_M);
  uint64_t* full = bars;                  // [STAGES] count AR_DEQUANT
  uint64_t* empty = full + G::STAGES;     // [STAGES] commit
  uint64_t* s_full = empty + G::STAGES;   // [tile & 1] commit, and the tile's scales
  uint64_t* p_full = s_full + 2;          // [tile & 1] count AR_SOFTMAX
  uint64_t* pv_done = p_full + 2;         // [tile & 1] commit
  uint64_t* q_full = pv_done + 2;         // count AR_SOFTMAX
  uint64_t* sum_done = q_full + 1;      // [32 rows] count 2: both groups' sums are there
  uint64_t* drained = sum_done + 4;       // commit
  uint64_t* raw_full = drained + 1;       // [RAWS] the copy
  uint64_t* raw_empty = raw_full + G::RAWS;  // [RAWS] count AR_DEQUANT
  int* raw_rows = reinterpret_cast<int*>(raw_empty + G::RAWS);  // [RAWS] positions in the stage
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(raw_rows + G::RAWS);
  static_assert((2 * G::STAGES + 12 + 2 * G::RAWS) * 8 + 4 * G::RAWS + 4 <= 512, "barriers");
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  if (warp == AR_SOFTMAX + AR_DEQUANT) tmem_alloc(tmem_slot, G::COLS);
  if (threadIdx.x == 0) {
    for (int i = 0; i < G::STAGES; i++) {
      mbar_init(&full[i], AR_DEQUANT);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; i++) {
      mbar_init(&s_full[i], 2);
      mbar_init(&p_full[i], AR_SOFTMAX);
      mbar_init(&pv_done[i], 1);
    }
    mbar_init(q_full, AR_SOFTMAX);
    for (int i = 0; i < 4; i++) {
      mbar_init(&sum_done[i], 2);
    }
    mbar_init(drained, 1);
    for (int i = 0; i < G::RAWS; i++) {
      mbar_init(&raw_full[i], 1);
      mbar_init(&raw_empty[i], AR_DEQUANT);
    }
    fence_mbar_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_launch_dependents();  // after the allocation: the next kernel's cannot come between
  pdl_wait();

  const int total = ArList::total(a), ctas = min(a.ctas, total);
  const bool busy = (int)blockIdx.x < ctas;
  const int first = busy ? ArList::first_of(blockIdx.x, total, ctas) : 0;
  const int last = busy ? ArList::first_of(blockIdx.x + 1, total, ctas) : 0;
  bool ok = true;

  if (!busy) {
    // nothing to do but to give the TMEM back
    if (threadIdx.x == 0) a.joints[blockIdx.x].parts = 0;
  } else if (warp < AR_SOFTMAX) {
    // ---------------- softmax: thread = row ----------------
    const int group = warp / AR_GROUP, quarter = warp % AR_GROUP, row = threadIdx.x % AR_M;
    const uint32_t lanes = tmem + ((uint32_t)(32 * quarter) << 16);
    const int rows = a.n * a.group;
    ArRun run;
    run.begin(a, first, last);
    int tile = 0, runs = 0, met = 0;  // of the CTA
    do {
      const int r = run.at.mb * AR_M + row;  // row of the unit's head
      const int i = r / a.group;
      // Q: the row in fp16, 16 dimensions in 8 columns; a half of it by each group. bf16: times a power of two of the
      // row's own (q_shift), whose inverse its thread multiplies the scores with. Padding counts as 0.
      const int r_load = i < run.at.span.count ? r : rows;
      int shift = 0;
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        float amax = 0.f;
#pragma unroll 4
        for (int d = 0; d < D; d += 8) {
          float f[8];
          q8_values<T>(load_q8<T>(a, run.at.b, run.at.kh, r_load, d), f);
#pragma unroll
          for (int e = 0; e < 8; e++) amax = fmaxf(amax, fabsf(f[e]));
        }
        shift = q_shift(amax);
      }
      const float up = (a.scale < 0.f ? -1.f : 1.f) * exp2_int(shift);
      const float factor = fabsf(a.scale) * 1.4426950408889634f * exp2_int(-shift);  // fp16: with the keys' scales
      const f32x2 factor2 = pair(factor, factor);
#pragma unroll 1
      for (int c = group * (D / 128); c < (group + 1) * (D / 128); c++) {
        uint32_t w[32];
#pragma unroll
        for (int d = 0; d < 64; d += 8) {
          float f[8];
          q8_values<T>(load_q8<T>(a, run.at.b, run.at.kh, r_load, 64 * c + d), f);
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const __half2 h = __floats2half2_rn(f[2 * e] * up, f[2 * e + 1] * up);
            w[d / 2 + e] = *reinterpret_cast<const uint32_t*>(&h);
          }
        }
        tmem_st32(lanes + G::Q + 32 * c, w);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);

      const int run0 = tile;  // the run's first tile

      float ref = -INFINITY, sum = 0.f;  // of the row; the sum of this group's half
      bool wide = false;  // the run has met a scale outside 2^-40 .. 2^40: the sum is relative to its `mores`, else to 2^ref
      for (; tile < run0 + run.len; tile++) {
        const int p0 = (run.at.tile + tile - run0) * AR_TILE + group * AR_HALF;
        ok = warp_wait(&s_full[tile & 1], (uint32_t)((tile / 2) & 1), a.err);
        if (!ok) break;
        tc_fence_after();
        const float* ks = scales + ((tile & 1) * 2 + group) * AR_SCALES;
        const uint32_t scores = lanes + G::S + (tile & 1) * AR_TILE + group * AR_HALF;
        // The run's first tile with a scale outside 2^-40 .. 2^40: from here on the sum follows the largest weight. (Both
        // groups have met in this tile, so the other one has read the `mores` of the run before.)
        auto turn = [&]() {
          if (!wide && reinterpret_cast<const uint32_t*>(ks)[3 * AR_HALF + 1]) {
            wide = true;
            mores[group * AR_M + row] = ref == -INFINITY ? make_float2(0.f, -INFINITY) : make_float2(ref, 0.f);
          }
        };
        uint32_t s[AR_HALF];
        tmem_ld32(scores, s);
        tmem_wait_ld();

        // t = ks * s + log2 vs, and the row's maximum over both halves
        f32x2 t[AR_HALF / 2];
#pragma unroll
        for (int e = 0; e < AR_HALF; e += 4) {
          const ulonglong2 k4 = *reinterpret_cast<const ulonglong2*>(ks + e);
          const ulonglong2 v4 = *reinterpret_cast<const ulonglong2*>(ks + AR_HALF + e);
          f32x2 x = pair(__uint_as_float(s[e]), __uint_as_float(s[e + 1]));
          f32x2 y = pair(__uint_as_float(s[e + 2]), __uint_as_float(s[e + 3]));
          if constexpr (std::is_same<T, __nv_bfloat16>::value) {
            x = mul2(x, factor2);
            y = mul2(y, factor2);
          }
          t[e / 2] = fma2(x, k4.x, v4.x);
          t[e / 2 + 1] = fma2(y, k4.y, v4.y);
        }
        if (p0 + AR_HALF > min(run.at.span.base, run.at.span.len)) {  // the same for all threads
          const uint32_t see = (uint32_t)ar_visible(a, run.at.b, run.at.span, i, p0);
#pragma unroll
          for (int e = 0; e < AR_HALF / 2; e++) {
            const float2 x = halves(t[e]);
            t[e] = pair(see >> 2 * e & 1 ? x.x : -INFINITY, see >> (2 * e + 1) & 1 ? x.y : -INFINITY);
          }
        }
        float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < AR_HALF / 2; e++) {
          const float2 x = halves(t[e]);
          m[e % 4] = fmaxf(fmaxf(m[e % 4], x.x), x.y);
        }
        float top = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
        float* mine = tops + (tile & 1) * 2 * AR_M + row;
        mine[group * AR_M] = top;
        ar_meet(quarter);
        met++;
        top = fmaxf(top, mine[(1 - group) * AR_M]);
        const bool grow = top > ref + 8.f || (ref == -INFINITY && top > ref);
        if (__any_sync(0xffffffffu, grow)) {
          const float next = grow ? top : ref;
          const float f = ref == next || ref == -INFINITY ? 1.f : exp2_approx(ref - next);  // no weight yet: 0, or NaN
          turn();
          if (!wide) sum *= f;
          if (tile > run0) {
            // O holds this unit's tiles so far: wait for the last of them and rescale it, each group half its columns
            ok = warp_wait(&pv_done[(tile - 1) & 1], (uint32_t)(((tile - 1) / 2) & 1), a.err);
            if (!ok) break;
            tc_fence_after();
#pragma unroll 1
            for (int c = group * (D / 2); c < (group + 1) * (D / 2); c += 32) {
              uint32_t o[32];
              tmem_ld32(lanes + G::O + c, o);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tmem_st32(lanes + G::O + c, o);
            }
            tmem_wait_st();
          }
          ref = next;
        }

        // weights 2^(t - ref + 6), at most 2^14, in fp16; and the sum of the unrounded ones over their value scales
        const float lift = 6.f - (ref == -INFINITY ? 0.f : ref);
        const f32x2 lift2 = pair(lift, lift);
        f32x2 acc0 = pair(0.f, 0.f), acc1 = acc0;
        uint32_t w[AR_HALF / 2];
#pragma unroll
        for (int e = 0; e < AR_HALF / 2; e += 2) {
          float2 x = halves(add2(t[e], lift2)), y = halves(add2(t[e + 1], lift2));
          x = make_float2(exp2_approx(x.x), exp2_approx(x.y));
          y = make_float2(exp2_approx(y.x), exp2_approx(y.y));
          const ulonglong2 i4 = *reinterpret_cast<const ulonglong2*>(ks + 2 * AR_HALF + 2 * e);
          acc0 = fma2(pair(x.x, x.y), i4.x, acc0);
          acc1 = fma2(pair(y.x, y.y), i4.y, acc1);
          const __half2 h0 = __floats2half2_rn(x.x, x.y), h1 = __floats2half2_rn(y.x, y.y);
          w[e] = *reinterpret_cast<const uint32_t*>(&h0);
          w[e + 1] = *reinterpret_cast<const uint32_t*>(&h1);
        }
        const float2 added = halves(add2(acc0, acc1));
        const float before = sum;
        sum += added.x + added.y;
        const uint2 rare = *reinterpret_cast<const uint2*>(ks + 3 * AR_HALF);  // positions of scale 0; far scales
        if (rare.x | rare.y) {  // the same for all threads
#pragma unroll
          for (int e = 0; e < AR_HALF / 2; e++)
            w[e] &= (rare.x >> 2 * e & 1 ? 0u : 0xffffu) | (rare.x >> (2 * e + 1) & 1 ? 0u : 0xffff0000u);
          turn();
          if (wide) {
            // the sum by itself, from the scores again: weights without their values' scales
            const uint32_t see = (uint32_t)ar_visible(a, run.at.b, run.at.span, i, p0);
            const float from = ref == -INFINITY ? 0.f : ref;
            float2* more = mores + group * AR_M + row;
            float at = more->y + (more->x - from);
            sum = before;
#pragma unroll 1
            for (int c = 0; c < AR_HALF; c += 16) {
              uint32_t z[16];
              tmem_ld16(scores + c, z);
              float next = at;
#pragma unroll
              for (int e = 0; e < 16; e++) {
                float y = __uint_as_float(z[e]);
                if constexpr (std::is_same<T, __nv_bfloat16>::value) y *= factor;
                const float lv = ks[AR_HALF + c + e];  // t + lift as above, less lv; of scale 0 without it
                y = lv == -INFINITY ? y * ks[c + e] + lift : fmaf(y, ks[c + e], lv) + lift - lv;
                y = see >> (c + e) & 1 ? y : -INFINITY;
                next = fmaxf(next, y);
                z[e] = __float_as_uint(y);
              }
              if (at != next && at != -INFINITY) sum *= exp2_approx(at - next);
              at = next;
              const float base = at == -INFINITY ? 0.f : at;
#pragma unroll
              for (int e = 0; e < 16; e++) sum += exp2_approx(__uint_as_float(z[e]) - base);
            }
            *more = make_float2(from, at);
          }
        }
        tmem_st16(scores, w);  // over the first half of the scores that they come from
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[tile & 1]);
      }
      if (!ok) break;

      // ---- the unit's (or its part's) result: the columns' halves by the two groups ----
      const int end = tile - 1;  // the run's last tile
      sums[group * AR_M + row] = sum;
      __syncwarp();
      if (lane == 0) mbar_arrive(&sum_done[quarter]);
      ok = warp_wait(&sum_done[quarter], (uint32_t)(runs++ & 1), a.err) &&
           warp_wait(&pv_done[end & 1], (uint32_t)((end / 2) & 1), a.err);
      if (!ok) break;
      sum = sums[row] + sums[AR_M + row];
      float more = 0.f;
      if (wide) {  // relative to the same ref by now
        const float2 m0 = mores[row], m1 = mores[AR_M + row];
        more = fmaxf(m0.y, m1.y);
        if (more == -INFINITY) {  // nothing seen
          more = 0.f;
        } else {
          sum = shrunk(sums[row], m0.y - more) + shrunk(sums[AR_M + row], m1.y - more);
          ref = m0.x + more;
        }
      }
      tc_fence_after();
      const int slot = 2 * blockIdx.x + (run.t == first ? 0 : 1);
      const bool live = r < rows;
      const bool none = sum == 0.f || i >= run.at.span.count;
      // (root to be multiplied with twice: its square may be outside of fp32's range)
      const float inv = none ? 0.f : 1.f / sum, root = exp2_approx(-0.5f * more);
      float* part = a.part + ((int64_t)slot * AR_M + row) * D;
#pragma unroll 1
      for (int c = group * (D / 2); c < (group + 1) * (D / 2); c += 32) {
        uint32_t o[32];
        tmem_ld32(lanes + G::O + c, o);
        tmem_wait_ld();
        if (!live) continue;
        if (run.whole) {
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            float f[8];
#pragma unroll
            for (int x = 0; x < 8; x++) f[x] = none ? 0.f : __uint_as_float(o[e + x]) * inv * root * root;
            store_row8<T>(a, run.at.b, run.at.kh, r, c + e, f);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            *reinterpret_cast<float4*>(part + c + e) =
                make_float4(__uint_as_float(o[e]) * root * root, __uint_as_float(o[e + 1]) * root * root,
                            __uint_as_float(o[e + 2]) * root * root, __uint_as_float(o[e + 3]) * root * root);
        }
      }
      if (live && !run.whole && group == 0)
        *reinterpret_cast<float2*>(a.stat + ((int64_t)slot * AR_M + row) * 2) = make_float2(ref, sum);
      tc_fence_before();  // the loads of O come before the next unit's products (through q_full)
    } while (run.next(a));
    for (; met < last - first; met++) ar_meet(quarter);
  } else if (warp < AR_SOFTMAX + AR_DEQUANT) {
    // ---------------- dequantise ----------------
    // A warp takes whole rows (D = 256: one, a lane 8 codes; D = 128: two), 8 codes becoming one 16-byte chunk of the
    // swizzled row. Rows of one lane differ by multiples of 8, so its swizzle is a constant.
    const int w = warp - AR_SOFTMAX;
    constexpr int LPR = D / 8;               // lanes per row
    constexpr int RPW = 32 / LPR;            // rows per warp and step
    constexpr int STEPS = AR_TILE / (8 * RPW);
    const int row = w * RPW + lane / LPR, chunk = lane % LPR;  // + 8 RPW per step
    const uint32_t dst = (uint32_t)(chunk / 8 * (AR_TILE * 128) + row * 128 + ((chunk % 8) ^ (row & 7)) * 16);
    const int items = 2 * (last - first);
    int stage = 0, use = 0, rs = 0, ruse = 0;
    for (int it = 0; it < items; it++) {
      ok = warp_wait(&raw_full[rs], (uint32_t)(ruse & 1), a.err);
      if (!ok) break;
      const uint8_t* src = raw + rs * G::RAW + row * D + chunk * 8;
      uint2 c[STEPS];
#pragma unroll
      for (int i = 0; i < STEPS; i++) c[i] = *reinterpret_cast<const uint2*>(src + i * 8 * RPW * D);
      const int there = raw_rows[rs] - row;  // rows past the sequence's end: zeros
      if (raw_rows[rs] < AR_TILE) {
#pragma unroll
        for (int i = 0; i < STEPS; i++)
          if (i * 8 * RPW >= there) c[i] = make_uint2(0u, 0u);
      }
      if (use > 0) {
        ok = warp_wait(&empty[stage], (uint32_t)((use - 1) & 1), a.err);
        if (!ok) break;
      }
      uint8_t* p = smem + stage * G::ITEM + dst;
#pragma unroll
      for (int i = 0; i < STEPS; i++) {
        uint4 v;
        codes_to_half2<FMT>(c[i].x, v.x, v.y);
        codes_to_half2<FMT>(c[i].y, v.z, v.w);
        *reinterpret_cast<uint4*>(p + i * 8 * RPW * 128) = v;
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&full[stage]);
        mbar_arrive(&raw_empty[rs]);
      }
      if (++stage == G::STAGES) stage = 0, use++;
      if (++rs == G::RAWS) rs = 0, ruse++;
    }
  } else {
    ArRun run;
    if (warp < AR_SOFTMAX + AR_DEQUANT + 3) run.begin(a, first, last);
    if (warp == AR_SOFTMAX + AR_DEQUANT) {
      // ---------------- issue the products: one warp, one of its lanes. All values are the warp's (broadcast where
      // the compiler cannot see it), so that operands and descriptors are built in uniform registers: with one lane's
      // own values the issue of a tile's products took 2300 cycles, longer than the products ----------------
      if (lane == 0) ArList::note(a, blockIdx.x, first, run.at, total, ctas);
      const bool leader = elect_one();
      int stage = 0, use = 0, tile = 0, runs = 0;
      const uint32_t items = smem_u32(smem), tm = __shfl_sync(0xffffffffu, tmem, 0);
      auto wait = [&](uint64_t* bar, int parity) {
        return __all_sync(0xffffffffu, ar_wait(bar, (uint32_t)(parity & 1), a.err)) != 0;
      };
      // S of the CTA's tile t, where the weights of tile t - 2 were
      auto scores = [&](int t) {
        ok = wait(&full[stage], use) && (t < 2 || wait(&pv_done[t & 1], t / 2 - 1));
        if (!ok) return;
        tc_fence_after();
        const uint32_t b = ar_k_major(items + stage * G::ITEM), d = tm + G::S + (t & 1) * AR_TILE;
        if (leader) {
#pragma unroll
          for (int k = 0; k < D / 16; k++)
            tc_mma_f16_ts(d, tm + G::Q + 8 * k, ar_desc(b + k / 4 * (AR_TILE * 128 / 16) + k % 4 * 2),
                                ar_idesc(AR_TILE, false), k != 0);
          tc_commit(&empty[stage]);
          tc_commit(&s_full[t & 1]);
        }
        __syncwarp();
        if (++stage == G::STAGES) stage = 0, use++;
      };
      bool more = true;
      while (more) {
        const int len = __shfl_sync(0xffffffffu, run.len, 0);
        ok = wait(q_full, runs++);
        if (!ok) break;
        scores(tile);
        if (ok && len > 1) scores(tile + 1);
        for (int j = 0; j < len && ok; j++, tile++) {
          ok = wait(&full[stage], use) && wait(&p_full[tile & 1], tile / 2);
          if (!ok) break;
          tc_fence_after();
          const uint32_t b = ar_mn_major(items + stage * G::ITEM, AR_TILE * 128), p = tm + G::S + (tile & 1) * AR_TILE;
          if (leader) {
#pragma unroll
            for (int k = 0; k < AR_TILE / 16; k++)  // (weights of 32 positions in 16 columns, the others' 32 columns on)
              tc_mma_f16_ts(tm + G::O, p + k / 2 * AR_HALF + k % 2 * 8, ar_desc(b + k * (2048 / 16)),
                                  ar_idesc(D, true), (j | k) != 0);
            tc_commit(&empty[stage]);
            tc_commit(&pv_done[tile & 1]);
          }
          __syncwarp();
          if (++stage == G::STAGES) stage = 0, use++;
          if (j + 2 < len) scores(tile + 2);
        }
        more = __all_sync(0xffffffffu, ok && run.next(a)) != 0;
      }
      // nothing may still write TMEM when it is given back
      if (leader) tc_commit(drained);
      __syncwarp();
      ar_wait(drained, 0, a.err);
    } else if (warp == AR_SOFTMAX + AR_DEQUANT + 1 && lane == 0) {
      // ---------------- copy the codes: one thread; items in the order K0, K1, V0, K2, V1, .. of each run --------
      int rs = 0, ruse = 0, kpos = 0, vpos = 0;
      const int items = 2 * (last - first);
      for (int it = 0; it < items; it++) {
        if (ruse > 0) {
          ok = ar_wait(&raw_empty[rs], (uint32_t)((ruse - 1) & 1), a.err);
          if (!ok) break;
        }
        const bool key = kpos < run.len && kpos - vpos < 2;
        const int p0 = (run.at.tile + (key ? kpos++ : vpos++)) * AR_TILE, n = min(run.at.span.len - p0, AR_TILE);
        raw_rows[rs] = n;
        mbar_arrive_expect_tx(&raw_full[rs], n * D);
        bulk_g2s(raw + rs * G::RAW, (key ? a.kc : a.vc) + (((int64_t)run.at.b * a.kv + run.at.kh) * a.cap + p0) * D, n * D,
                 &raw_full[rs]);
        if (++rs == G::RAWS) rs = 0, ruse++;
        if (vpos == run.len && it + 1 < items) {
          run.next(a);
          kpos = vpos = 0;
        }
      }
      // no copy may still be under way when the CTA ends (after a wait that gave up, one may be)
      for (int i = 0; i < G::RAWS; i++) {
        const int uses = ruse + (i < rs ? 1 : 0);
        if (uses > 0) ar_wait(&raw_full[i], (uint32_t)((uses - 1) & 1), a.err);
      }
    } else if (warp == AR_SOFTMAX + AR_DEQUANT + 2) {
      // ---------------- the tiles' scales: two positions a lane, loaded a tile ahead ----------------
      const float factor =
          std::is_same<T, __half>::value ? fabsf(a.scale) * 1.4426950408889634f : 1.f;  // bf16: a row's own, later
      float k[2], v[2];
      int j = 0;
      bool wide = false;  // the run has met a scale outside 2^-40 .. 2^40
      auto load = [&]() {
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const int p = (run.at.tile + j) * AR_TILE + h * AR_HALF + lane;
          const bool in = p < run.at.span.len;
          const int64_t at = ((int64_t)run.at.b * a.kv + run.at.kh) * a.cap + p;
          k[h] = in ? a.ks[at] : 0.f;
          v[h] = in ? a.vs[at] : 0.f;
        }
      };
      load();
      for (int t = 0; t < last - first; t++) {
        wide = wide || __any_sync(0xffffffffu, far_scale(v[0]) || far_scale(v[1]));
        ArScales made;  // before the wait: what follows it is on the softmax's path
        made.set(k, v, factor, wide);
        if (t >= 2) {  // the softmax is through with tile t - 2
          ok = warp_wait(&pv_done[t & 1], (uint32_t)((t / 2 - 1) & 1), a.err);
          if (!ok) break;
        }
        made.store(scales + (t & 1) * 2 * AR_SCALES, wide);
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_full[t & 1]);
        if (++j == run.len) {
          j = 0;
          wide = false;
          if (!run.next(a)) break;
        }
        load();
      }
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == AR_SOFTMAX + AR_DEQUANT) tmem_dealloc(tmem, G::COLS);
}

}  // namespace gsq
