// Penalties, biases and a grammar's mask on rows of logits, and the token of
// the highest result (gsq_adjust_logits); the token history behind the
// penalties (gsq_record_tokens).
//
// Every step is rounded to fp32 on its own (no fused multiply-add), so the
// result is the formula's in any order of evaluation a host would use, and
// ties go to the lowest token.
//
// Bound: HBM bytes, one read and one write of the rows.  A row belongs to one
// cluster of up to 8 CTAs, each with a run of its tokens: one launch, in which
// the CTAs' best tokens meet in distributed shared memory.  A thread takes
// eight tokens at a time, as two 16-byte pieces where every row starts on such
// a boundary, copied LG_STAGES - 1 steps ahead through shared memory (each
// thread its own, so no barrier), else one by one in neighbouring lanes, one
// step ahead in registers; the masks of the CTA's run are in shared memory from
// the start.  That pass streams: it leaves the few tokens that the penalties or
// a bias concern (some thousand of 248320) as they are, and out of the maximum.
// A second pass gathers them from the bit masks into a queue for each warp and
// works on them lane by lane, so that the scattered reads of their counts wait
// together and not one after the other in the stream.  A token's biases are
// added in list order by the thread that has the token: no atomic orders a sum.
// Measured with penalties, 100 biases and a mask: 64 rows of 248320 fp32
// 37 us (131 MB, 3.6 TB/s), one row 12 us.
#include <atomic>
#include <cstdio>

#include "gsq_common.cuh"
#include "gsq_host.h"
#include "../../include/gsq_model.h"

using namespace gsq;

namespace {

constexpr int LG_THREADS = 512;           // of a CTA, at most
constexpr int LG_QUEUE = 256;             // tokens of a warp's queue
constexpr int LG_STAGES = 4;              // of a thread's eight tokens, on their way
constexpr int LG_CLUSTER = 8;             // CTAs of a row, at most
constexpr int64_t LG_VOCAB = 1ll << 20;   // tokens at most: 2^17 a CTA, whose masks fit its shared memory

struct LogitsArgs {
  const void* logits;
  int64_t row_stride, vocab, words;
  int cluster, run;  // CTAs of a row, tokens of each (a multiple of 128)
  int32_t* seen;    // [rows, words] or null
  int32_t* counts;  // [rows, vocab]
  const float *repetition, *frequency, *presence;  // [rows] or null
  const int32_t* bias_ids;                         // [rows, biases]
  const float* bias_values;
  int64_t biases;
  const int32_t* allowed;  // row r's words at r * allowed_stride
  int64_t allowed_stride;
  float* out;
  int32_t* next;
  int record;
};

// Orders floats as unsigned integers; NaN above everything, -0 as +0.
__device__ __forceinline__ uint32_t order_key(float z) {
  if (isnan(z)) return 0xffffffffu;
  const uint32_t u = __float_as_uint(z + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ unsigned long long warp_max(unsigned long long k) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const unsigned long long p = __shfl_xor_sync(0xffffffffu, k, o);
    k = p > k ? p : k;
  }
  return k;
}

// The history of row r learns token v (bit and, for a generated token, count).
__device__ __forceinline__ void remember(int32_t* seen, int32_t* counts, int64_t words, int64_t vocab, int64_t r,
                                         int64_t v, bool generated) {
  atomicOr(seen + r * words + (v >> 5), (int32_t)(1u << (v & 31)));
  if (generated) atomicAdd(counts + r * vocab + v, 1);
}

// BYTES (8 or 16) of global memory to shared memory, asynchronously.
template <int BYTES>
__device__ __forceinline__ void cp_async(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(dst)), "l"(src), "n"(BYTES) : "memory");
}

__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// VEC: the rows of logits and out start on 16-byte (two-byte types: 8-byte) boundaries, and vocab % 4 == 0.
// Dynamic shared memory: the masks of the CTA's run (tokens that the second pass finishes, allowed tokens), the warps'
// queues, and with VEC the stages.
template <typename T, bool VEC>
__global__ void __launch_bounds__(LG_THREADS) adjust_kernel(const LogitsArgs a) {
  extern __shared__ __align__(16) uint32_t smem[];
  __shared__ unsigned long long part[LG_THREADS / 32], cta_best;
  pdl_launch_dependents();
  pdl_wait();
  const int64_t row = blockIdx.y;
  const int vocab = (int)a.vocab, lo = blockIdx.x * a.run, hi = min(vocab, lo + a.run);
  const int tid = threadIdx.x, lane = tid & 31, threads = blockDim.x, words = (max(hi - lo, 0) + 31) / 32;
  uint32_t *late_mask = smem, *allowed_mask = smem + a.run / 32;
  uint32_t* queue = smem + a.run / 16 + (tid >> 5) * LG_QUEUE;
  const T* x = static_cast<const T*>(a.logits) + row * a.row_stride;
  float* out = a.out + row * vocab;
  const int32_t* seen_row = a.seen ? a.seen + row * a.words : nullptr;
  const int32_t* ids = a.biases ? a.bias_ids + row * a.biases : nullptr;
  const int biases = (int)a.biases;

  // Eight tokens a step. token(v0, e): token e of this thread in the step that begins with v0.
  const int step = 8 * threads;
  auto token = [&](int v0, int e) { return VEC ? v0 + e / 4 * (4 * threads) + 4 * tid + e % 4 : v0 + e * threads + tid; };
  constexpr int PIECE = 4 * sizeof(T);  // bytes of a copied piece
  uint8_t* ring = reinterpret_cast<uint8_t*>(smem + a.run / 16 + threads / 32 * LG_QUEUE);
  T next[VEC ? 1 : 8];
  int ahead = lo, put = 0;
  auto load = [&]() {  // the step `ahead`
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const int v = token(ahead, 4 * i);
        if (v < hi) cp_async<PIECE>(ring + ((put * 2 + i) * threads + tid) * PIECE, x + v);
      }
      cp_async_commit();
      put = put + 1 == LG_STAGES ? 0 : put + 1;
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++)
        if (token(ahead, e) < hi) next[e] = x[token(ahead, e)];
    }
    ahead += step;
  };
#pragma unroll
  for (int i = 0; i < (VEC ? LG_STAGES - 1 : 1); i++) load();

  for (int w = tid; w < words; w += threads) {
    late_mask[w] = seen_row ? (uint32_t)seen_row[(lo >> 5) + w] : 0u;  // lo % 32 == 0
    allowed_mask[w] = a.allowed ? (uint32_t)a.allowed[row * a.allowed_stride + (lo >> 5) + w] : ~0u;
  }
  if (biases) {
    __syncthreads();
    for (int i = tid; i < biases; i += threads) {
      const int id = ids[i];
      if (id >= lo && id < hi) atomicOr(&late_mask[(id - lo) >> 5], 1u << (id & 31));
    }
  }
  __syncthreads();

  unsigned long long best = 0;
  float top = -INFINITY;  // the thread's best so far
  int top_at = -1, get = 0;
  for (int v0 = lo; v0 < hi; v0 += step) {
    alignas(16) T raw[8];
    if constexpr (VEC) {
      load();
      cp_async_wait<LG_STAGES - 1>();
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const uint8_t* p = ring + ((get * 2 + i) * threads + tid) * PIECE;
        if constexpr (PIECE == 16) reinterpret_cast<uint4*>(raw)[i] = *reinterpret_cast<const uint4*>(p);
        else reinterpret_cast<uint2*>(raw)[i] = *reinterpret_cast<const uint2*>(p);
      }
      get = get + 1 == LG_STAGES ? 0 : get + 1;
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) raw[e] = next[e];
      load();
    }
    alignas(16) float z[8];
#pragma unroll
    for (int e = 0; e < 8; e++) z[e] = token(v0, e) < hi ? to_f32(raw[e]) : -INFINITY;
    uint32_t late = 0, hidden = 0;  // bit e: for the second pass, not allowed
#pragma unroll
    for (int i = 0; i < (VEC ? 2 : 8); i++) {
      constexpr int N = VEC ? 4 : 1;
      const int v = token(v0, i * N);
      if (v < hi) {
        late |= (late_mask[(v - lo) >> 5] >> (v & 31) & ((1u << N) - 1)) << i * N;
        hidden |= (~allowed_mask[(v - lo) >> 5] >> (v & 31) & ((1u << N) - 1)) << i * N;
      }
    }
    hidden &= ~late;
    if (hidden) {
#pragma unroll
      for (int e = 0; e < 8; e++) z[e] = hidden >> e & 1 ? -INFINITY : z[e];
    }
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < 2; i++)
        if (token(v0, 4 * i) < hi)
          *reinterpret_cast<float4*>(out + token(v0, 4 * i)) = *reinterpret_cast<const float4*>(z + 4 * i);
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++)
        if (token(v0, e) < hi) out[token(v0, e)] = z[e];
    }
    // the thread's best token: they rise with e, and those past the end are -inf and come after the others
    if (late) {
#pragma unroll
      for (int e = 0; e < 8; e++) z[e] = late >> e & 1 ? -INFINITY : z[e];
    }
    float m = z[0];
    bool nan = isnan(z[0]);
#pragma unroll
    for (int e = 1; e < 8; e++) {
      m = fmaxf(m, z[e]);
      nan = nan || isnan(z[e]);
    }
    if (nan) {
      int at = 0;
#pragma unroll
      for (int e = 7; e >= 0; e--) at = isnan(z[e]) ? e : at;
      const unsigned long long k = 0xffffffffull << 32 | (uint32_t)~(uint32_t)token(v0, at);
      best = k > best ? k : best;
    } else if (m > top || top_at < 0) {
      int at = 0;
#pragma unroll
      for (int e = 7; e >= 0; e--) at = z[e] == m ? e : at;
      if (token(v0, at) < hi) {
        top = m;
        top_at = token(v0, at);
      }
    }
  }
  if (top_at >= 0) {
    const unsigned long long k = (unsigned long long)order_key(top) << 32 | (uint32_t)~(uint32_t)top_at;
    best = k > best ? k : best;
  }
  if (biases || seen_row) {
    __syncthreads();  // the values are written
    const float* val = biases ? a.bias_values + row * a.biases : nullptr;
    const float rep = a.repetition ? a.repetition[row] : 1.f;
    const float freq = a.frequency ? a.frequency[row] : 0.f;
    const float pres = a.presence ? a.presence[row] : 0.f;
    int queued = 0;
    auto finish = [&]() {
      __syncwarp();
      for (int i0 = 0; i0 < queued; i0 += 32) {
        const bool mine = i0 + lane < queued;
        const int v = mine ? (int)queue[i0 + lane] : -1;
        float y = mine ? out[v] : 0.f;
        if (mine && seen_row && (uint32_t)seen_row[v >> 5] >> (v & 31) & 1u) {
          const int32_t n = a.counts[row * vocab + v];
          y = y > 0.f ? __fdiv_rn(y, rep) : __fmul_rn(y, rep);
          if (n > 0) {
            y = __fsub_rn(y, __fmul_rn(freq, (float)n));
            y = __fsub_rn(y, pres);
          }
        }
        if (biases) {
          // the list against the warp's tokens, 32 entries at a time, each token's sum in the list's order
          float s = 0.f;
          bool any = false;
          for (int j0 = 0; j0 < biases; j0 += 32) {
            const int id = j0 + lane < biases ? ids[j0 + lane] : -1;
            const float b = j0 + lane < biases ? val[j0 + lane] : 0.f;
            unsigned here = __ballot_sync(0xffffffffu, id >= lo && id < hi);
            while (here) {
              const int l = __ffs(here) - 1;
              here &= here - 1;
              const float one = __shfl_sync(0xffffffffu, b, l);
              if (__shfl_sync(0xffffffffu, id, l) == v) {
                s = __fadd_rn(s, one);
                any = true;
              }
            }
          }
          if (any) y = __fadd_rn(y, s);
        }
        if (!mine) continue;
        if (!(allowed_mask[(v - lo) >> 5] >> (v & 31) & 1u)) y = -INFINITY;
        out[v] = y;
        const unsigned long long k = (unsigned long long)order_key(y) << 32 | (uint32_t)~(uint32_t)v;
        best = k > best ? k : best;
      }
      __syncwarp();
      queued = 0;
    };
    for (int w0 = (tid >> 5) * 32; w0 < words; w0 += threads) {
      const int w = w0 + lane;
      uint32_t bits = w < words ? late_mask[w] : 0u;
      if (w < words && hi - lo - 32 * w < 32) bits &= (1u << (hi - lo - 32 * w)) - 1;  // past the last token
      // eight tokens of each word at a time: at most a queue full
      while (__any_sync(0xffffffffu, bits)) {
        const int mine = min(__popc(bits), 8);
        int at = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int u = __shfl_up_sync(0xffffffffu, at, o);
          if (lane >= o) at += u;
        }
        const int all = __shfl_sync(0xffffffffu, at, 31);
        if (queued + all > LG_QUEUE) finish();
        at += queued - mine;
        for (int i = 0; i < mine; i++) {
          queue[at + i] = lo + 32 * w + __ffs(bits) - 1;
          bits &= bits - 1;
        }
        queued += all;
      }
    }
    finish();
  }
  best = warp_max(best);
  if (lane == 0) part[tid >> 5] = best;
  __syncthreads();
  if (tid < 32) {
    best = warp_max(tid < blockDim.x / 32 ? part[tid] : 0ull);
    if (tid == 0) cta_best = best;
  }
  if (a.cluster > 1) cluster_sync_all();
  if (blockIdx.x == 0 && tid == 0) {
    for (int r = 1; r < a.cluster; r++) {
      uint32_t remote;
      unsigned long long k;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(&cta_best)), "r"(r));
      asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(k) : "r"(remote) : "memory");
      best = k > best ? k : best;
    }
    const int32_t v = (int32_t)~(uint32_t)best;
    a.next[row] = v;
    if (a.record) remember(a.seen, a.counts, a.words, a.vocab, row, v, true);
  }
  if (a.cluster > 1) cluster_sync_all();  // no CTA leaves before its best token is read
}

__global__ void __launch_bounds__(256) record_kernel(const int32_t* tokens, int64_t stride, int64_t rows, int64_t n,
                                                     int64_t vocab, int64_t words, int32_t* seen, int32_t* counts,
                                                     int generated) {
  pdl_launch_dependents();
  pdl_wait();
  const int64_t total = rows * n;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / n, v = tokens[r * stride + i % n];
    if (v >= 0 && v < vocab) remember(seen, counts, words, vocab, r, v, generated != 0);
  }
}

int fail(int code, const char* msg) { return set_last_error(code, msg); }

int launched(cudaError_t rc, const char* what) {
  if (rc == cudaSuccess) rc = cudaGetLastError();
  if (rc == cudaSuccess) return GSQ_OK;
  char buf[256];
  snprintf(buf, sizeof(buf), "%s: %s", what, cudaGetErrorString(rc));
  return fail(GSQ_ERR_CUDA, buf);
}

template <typename T, bool VEC>
cudaError_t adjust_launch(dim3 grid, cudaStream_t st, const LogitsArgs& a) {
  // where there are few CTAs, large ones (8 rows of 248320: 13.1 us, with 256 threads 17.5); many divide more evenly
  // when they are small (64 rows: 42 us, with 256 threads 37)
  const dim3 block(grid.x * grid.y <= 296 ? LG_THREADS : LG_THREADS / 2);
  const size_t smem = a.run / 4 + block.x / 32 * LG_QUEUE * 4 + (VEC ? LG_STAGES * block.x * 8 * sizeof(T) : 0);
  // (at most 2^17 tokens a CTA: 32 KB of masks)
  auto kernel = adjust_kernel<T, VEC>;
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64 || !(done.load(std::memory_order_relaxed) >> dev & 1)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 128 * 1024);
    if (e != cudaSuccess) return e;
    if (dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  return a.cluster > 1 ? launch_pdl_cluster(kernel, grid, block, a.cluster, st, smem, a)
                       : launch_pdl(kernel, grid, block, smem, st, a);
}

template <typename T>
cudaError_t adjust(bool vec, dim3 grid, cudaStream_t st, const LogitsArgs& a) {
  return vec ? adjust_launch<T, true>(grid, st, a) : adjust_launch<T, false>(grid, st, a);
}


}  // namespace

extern "C" {

int gsq_adjust_logits(const void* logits, int dtype, int64_t row_stride, int64_t rows, int64_t vocab, int32_t* seen,
                      int32_t* counts, const float* repetition, const float* frequency, const float* presence,
                      const int32_t* bias_ids, const float* bias_values, int64_t biases, const int32_t* allowed,
                      int64_t allowed_stride, float* out, int32_t* next, int record, gsq_stream_t stream) {
  if (dtype != DT_F32 && dtype != DT_F16 && dtype != DT_BF16) return fail(GSQ_ERR_ARG, "gsq_adjust_logits: bad dtype");
  if (rows < 0 || rows > 65535 || vocab <= 0 || vocab > LG_VOCAB || row_stride < vocab)
    return fail(GSQ_ERR_SIZE, "gsq_adjust_logits: bad shape");
  if (biases < 0 || biases > 65536) return fail(GSQ_ERR_SIZE, "gsq_adjust_logits: bad bias count");
  if (rows == 0) return GSQ_OK;
  if (!logits || !out || !next || (biases && (!bias_ids || !bias_values)))
    return fail(GSQ_ERR_ARG, "gsq_adjust_logits: null pointer");
  if (!seen != !counts) return fail(GSQ_ERR_ARG, "gsq_adjust_logits: seen and counts come together");
  if (!seen && (repetition || frequency || presence || record))
    return fail(GSQ_ERR_ARG, "gsq_adjust_logits: penalties and recording need a history");
  if (reinterpret_cast<uintptr_t>(logits) % (dtype == DT_F32 ? 4 : 2) ||
      !words_aligned({seen, counts, repetition, frequency, presence, bias_ids, bias_values, allowed, out, next}))
    return fail(GSQ_ERR_ALIGN, "gsq_adjust_logits: pointers not aligned to their type");
  LogitsArgs a = {};
  a.logits = logits;
  a.row_stride = row_stride;
  a.vocab = vocab;
  a.words = (vocab + 31) / 32;
  a.seen = seen;
  a.counts = counts;
  a.repetition = repetition;
  a.frequency = frequency;
  a.presence = presence;
  a.bias_ids = bias_ids;
  a.bias_values = bias_values;
  a.biases = biases;
  a.allowed = allowed;
  a.allowed_stride = allowed_stride;
  a.out = out;
  a.next = next;
  a.record = record;
  // 8 CTAs a row; fewer where there are more than run at once (four on an SM) and each would have under 6144 tokens
  // (us, with 8 / 4 / 2 CTAs a row: 256 rows of 248320 125 / 166 / 207, 512 rows of 32000 101 / 76 / 89).
  a.cluster = LG_CLUSTER;
  while (a.cluster > 1 && rows * a.cluster > 148 * 4 && vocab < 6144 * a.cluster) a.cluster /= 2;
  a.run = (int)((vocab + 128 * a.cluster - 1) / (128 * a.cluster) * 128);
  const dim3 grid((unsigned)a.cluster, (unsigned)rows);
  cudaStream_t st = (cudaStream_t)stream;
  const size_t size = dtype == DT_F32 ? 4 : 2;
  const bool vec = vocab % 4 == 0 && row_stride % 4 == 0 && reinterpret_cast<uintptr_t>(logits) % (4 * size) == 0 &&
                   reinterpret_cast<uintptr_t>(out) % 16 == 0;
  return launched(dtype == DT_F32   ? adjust<float>(vec, grid, st, a)
                  : dtype == DT_F16 ? adjust<__half>(vec, grid, st, a)
                                    : adjust<__nv_bfloat16>(vec, grid, st, a),
                  "gsq_adjust_logits");
}

int gsq_record_tokens(const int32_t* tokens, int64_t row_stride, int64_t rows, int64_t n, int64_t vocab, int32_t* seen,
                      int32_t* counts, int generated, gsq_stream_t stream) {
  if (rows < 0 || rows > 65535 || n < 0 || n > (1ll << 30) || vocab <= 0 || vocab > (1ll << 30) || row_stride < 0)
    return fail(GSQ_ERR_SIZE, "gsq_record_tokens: bad shape");
  if (rows == 0 || n == 0) return GSQ_OK;
  if (!tokens || !seen || !counts) return fail(GSQ_ERR_ARG, "gsq_record_tokens: null pointer");
  if (!words_aligned({tokens, seen, counts}))
    return fail(GSQ_ERR_ALIGN, "gsq_record_tokens: pointers not aligned to their type");
  const int64_t blocks = (rows * n + 255) / 256;
  return launched(launch_pdl(record_kernel, dim3((unsigned)(blocks < 148 * 8 ? blocks : 148 * 8)), dim3(256), 0,
                             (cudaStream_t)stream, tokens, row_stride, rows, n, vocab, (vocab + 31) / 32, seen, counts,
                             generated),
                  "gsq_record_tokens");
}

}  // extern "C"
