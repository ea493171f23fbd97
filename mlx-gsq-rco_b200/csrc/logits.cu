// Penalties, biases and a grammar's mask on rows of logits, and the token of
// the highest result (gsq_adjust_logits); the token history behind the
// penalties (gsq_record_tokens).
//
// Every step is rounded to fp32 on its own (no fused multiply-add), so the
// result is the formula's in any order of evaluation a host would use, and
// ties go to the lowest token.
//
// Bound: HBM bytes, one read and one write of the rows.  A row is cut into
// chunks of LG_CHUNK tokens, one CTA each, so that one row still fills the GPU
// (248320 tokens: 122 CTAs).  A thread holds eight tokens, as two 16-byte
// pieces where every row starts on such a boundary, else one by one in
// neighbouring lanes.  The penalties run only where a token's seen bit is set
// (some thousand of 248320 tokens), and only there the counts are read.  Biases
// of a chunk are gathered into shared memory first, duplicates summed in list
// order by one thread, so no atomic orders the sum.  Each CTA leaves its best
// token; a second launch (one warp per row) takes the best of them and
// records it.
#include <cstdio>

#include "gsq_common.cuh"
#include "gsq_host.h"
#include "../../include/gsq_model.h"

using namespace gsq;

namespace {

constexpr int LG_THREADS = 256;
constexpr int LG_CHUNK = 8 * LG_THREADS;  // tokens per CTA

struct LogitsArgs {
  const void* logits;
  int64_t row_stride, vocab, words, chunks;
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
  unsigned long long* best;  // [rows, chunks]
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

// Four tokens from v on, aligned for one load.
template <typename T>
__device__ __forceinline__ void load4(const T* p, float* f) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(f) = *reinterpret_cast<const float4*>(p);
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
    for (int i = 0; i < 4; i++) f[i] = to_f32(e[i]);
  }
}

// VEC: the rows of logits and out start on 16-byte (two-byte types: 8-byte) boundaries, and vocab % 4 == 0.
template <typename T, bool VEC>
__global__ void __launch_bounds__(LG_THREADS) adjust_kernel(const LogitsArgs a) {
  __shared__ __align__(16) float bias[LG_CHUNK];
  __shared__ unsigned long long part[LG_THREADS / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int64_t row = blockIdx.y;
  const int vocab = (int)a.vocab, c0 = blockIdx.x * LG_CHUNK;
  const int tid = threadIdx.x, lane = tid & 31;
  const T* x = static_cast<const T*>(a.logits) + row * a.row_stride;
  const int32_t* seen_row = a.seen ? a.seen + row * a.words : nullptr;
  const int32_t* allowed_row = a.allowed ? a.allowed + row * a.allowed_stride : nullptr;
  // token e of this thread, and its bits of the masks (bit e), one word for 4 tokens of 8 lanes or 1 of 32
  auto token = [&](int e) { return VEC ? c0 + e / 4 * (4 * LG_THREADS) + 4 * tid + e % 4 : c0 + e * LG_THREADS + tid; };
  alignas(16) float z[8] = {};
  uint32_t seen = 0, allowed = 0xffu;
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const int v = token(4 * i);
      if (v < vocab) {
        load4(x + v, z + 4 * i);
        if (seen_row) seen |= ((uint32_t)seen_row[v >> 5] >> (v & 31) & 15u) << 4 * i;
        if (allowed_row) allowed &= ((uint32_t)allowed_row[v >> 5] >> (v & 31) & 15u) << 4 * i | 15u << 4 * (1 - i);
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const int v = token(e);
      if (v < vocab) {
        z[e] = to_f32(x[v]);
        if (seen_row) seen |= ((uint32_t)seen_row[v >> 5] >> lane & 1u) << e;
        if (allowed_row && !((uint32_t)allowed_row[v >> 5] >> lane & 1u)) allowed &= ~(1u << e);
      }
    }
  }
  if (a.biases) {
#pragma unroll
    for (int i = 0; i < 2; i++) reinterpret_cast<float4*>(bias)[tid + i * LG_THREADS] = make_float4(0.f, 0.f, 0.f, 0.f);
    __syncthreads();
    const int32_t* ids = a.bias_ids + row * a.biases;
    const float* val = a.bias_values + row * a.biases;
    const int n = (int)a.biases;
    for (int i = tid; i < n; i += LG_THREADS) {
      const int id = ids[i];
      if (id < c0 || id - c0 >= LG_CHUNK || id >= vocab) continue;
      bool first = true;
      for (int j = 0; j < i && first; j++) first = ids[j] != id;
      if (!first) continue;
      float s = 0.f;
      for (int j = i; j < n; j++)
        if (ids[j] == id) s = __fadd_rn(s, val[j]);
      bias[id - c0] = s;
    }
    __syncthreads();
  }
  if (seen) {
    const float rep = a.repetition ? a.repetition[row] : 1.f;
    const float freq = a.frequency ? a.frequency[row] : 0.f;
    const float pres = a.presence ? a.presence[row] : 0.f;
#pragma unroll
    for (int e = 0; e < 8; e++) {
      if (seen >> e & 1) {
        float y = z[e];
        y = y > 0.f ? __fdiv_rn(y, rep) : __fmul_rn(y, rep);
        const int32_t n = a.counts[row * vocab + token(e)];
        if (n > 0) {
          y = __fsub_rn(y, __fmul_rn(freq, (float)n));
          y = __fsub_rn(y, pres);
        }
        z[e] = y;
      }
    }
  }
  if (a.biases) {
#pragma unroll
    for (int e = 0; e < 8; e++) z[e] = __fadd_rn(z[e], bias[token(e) - c0]);
  }
  if (allowed != 0xffu) {
#pragma unroll
    for (int e = 0; e < 8; e++) z[e] = allowed >> e & 1 ? z[e] : -INFINITY;
  }
  float* out = a.out + row * vocab;
  // the thread's best token: tokens rise with e, so those past the end come after the others
  if (c0 + LG_CHUNK > vocab) {
#pragma unroll
    for (int e = 0; e < 8; e++) z[e] = token(e) < vocab ? z[e] : -INFINITY;
  }
  float top = z[0];
  bool nan = isnan(z[0]);
#pragma unroll
  for (int e = 1; e < 8; e++) {
    top = fmaxf(top, z[e]);
    nan = nan || isnan(z[e]);
  }
  int at = 0;
  if (nan) {
#pragma unroll
    for (int e = 7; e >= 0; e--) at = isnan(z[e]) ? e : at;
    top = __int_as_float(0x7fffffff);
  } else {
#pragma unroll
    for (int e = 7; e >= 0; e--) at = z[e] == top ? e : at;
  }
  unsigned long long best = 0;
  if (token(at) < vocab) best = (unsigned long long)order_key(top) << 32 | (uint32_t)~(uint32_t)token(at);
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < 2; i++)
      if (token(4 * i) < vocab) *reinterpret_cast<float4*>(out + token(4 * i)) = *reinterpret_cast<const float4*>(z + 4 * i);
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++)
      if (token(e) < vocab) out[token(e)] = z[e];
  }
  best = warp_max(best);
  if (lane == 0) part[tid >> 5] = best;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < LG_THREADS / 32; w++) best = part[w] > best ? part[w] : best;
    a.best[row * a.chunks + blockIdx.x] = best;
  }
}

// The history of row r learns token v (bit and, for a generated token, count).
__device__ __forceinline__ void remember(int32_t* seen, int32_t* counts, int64_t words, int64_t vocab, int64_t r,
                                         int64_t v, bool generated) {
  atomicOr(seen + r * words + (v >> 5), (int32_t)(1u << (v & 31)));
  if (generated) atomicAdd(counts + r * vocab + v, 1);
}

__global__ void __launch_bounds__(32) pick_kernel(const LogitsArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const int64_t row = blockIdx.x;
  unsigned long long best = 0;
  for (int64_t i = threadIdx.x; i < a.chunks; i += 32) {
    const unsigned long long k = a.best[row * a.chunks + i];
    best = k > best ? k : best;
  }
  best = warp_max(best);
  if (threadIdx.x == 0) {
    const int32_t v = (int32_t)~(uint32_t)best;
    a.next[row] = v;
    if (a.record) remember(a.seen, a.counts, a.words, a.vocab, row, v, true);
  }
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

template <typename T>
cudaError_t adjust_launch(bool vec, dim3 grid, cudaStream_t st, const LogitsArgs& a) {
  return vec ? launch_pdl(adjust_kernel<T, true>, grid, dim3(LG_THREADS), 0, st, a)
             : launch_pdl(adjust_kernel<T, false>, grid, dim3(LG_THREADS), 0, st, a);
}

int64_t chunks_of(int64_t vocab) { return (vocab + LG_CHUNK - 1) / LG_CHUNK; }
bool al4(const void* p) { return reinterpret_cast<uintptr_t>(p) % 4 == 0; }

}  // namespace

extern "C" {

size_t gsq_adjust_logits_workspace_size(int64_t rows, int64_t vocab) {
  if (rows <= 0 || vocab <= 0) return 0;
  return (size_t)rows * chunks_of(vocab) * sizeof(unsigned long long);
}

int gsq_adjust_logits(const void* logits, int dtype, int64_t row_stride, int64_t rows, int64_t vocab, int32_t* seen,
                      int32_t* counts, const float* repetition, const float* frequency, const float* presence,
                      const int32_t* bias_ids, const float* bias_values, int64_t biases, const int32_t* allowed,
                      int64_t allowed_stride, float* out, int32_t* next, int record, void* workspace,
                      size_t workspace_bytes, gsq_stream_t stream) {
  if (dtype != DT_F32 && dtype != DT_F16 && dtype != DT_BF16) return fail(GSQ_ERR_ARG, "gsq_adjust_logits: bad dtype");
  if (rows < 0 || rows > 65535 || vocab <= 0 || vocab > (1ll << 30) || row_stride < vocab)
    return fail(GSQ_ERR_SIZE, "gsq_adjust_logits: bad shape");
  if (biases < 0 || biases > 65536) return fail(GSQ_ERR_SIZE, "gsq_adjust_logits: bad bias count");
  if (rows == 0) return GSQ_OK;
  if (!logits || !out || !next || (biases && (!bias_ids || !bias_values)))
    return fail(GSQ_ERR_ARG, "gsq_adjust_logits: null pointer");
  if (!seen != !counts) return fail(GSQ_ERR_ARG, "gsq_adjust_logits: seen and counts come together");
  if (!seen && (repetition || frequency || presence || record))
    return fail(GSQ_ERR_ARG, "gsq_adjust_logits: penalties and recording need a history");
  if (reinterpret_cast<uintptr_t>(logits) % (dtype == DT_F32 ? 4 : 2) || !al4(out) || !al4(next))
    return fail(GSQ_ERR_ALIGN, "gsq_adjust_logits: pointers not aligned to their type");
  if (!workspace || workspace_bytes < gsq_adjust_logits_workspace_size(rows, vocab))
    return fail(GSQ_ERR_WORKSPACE, "gsq_adjust_logits: workspace missing or too small");
  if (reinterpret_cast<uintptr_t>(workspace) % 8) return fail(GSQ_ERR_ALIGN, "gsq_adjust_logits: workspace not 8-byte aligned");
  LogitsArgs a = {};
  a.logits = logits;
  a.row_stride = row_stride;
  a.vocab = vocab;
  a.words = (vocab + 31) / 32;
  a.chunks = chunks_of(vocab);
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
  a.best = static_cast<unsigned long long*>(workspace);
  a.record = record;
  cudaStream_t st = (cudaStream_t)stream;
  const dim3 grid((unsigned)a.chunks, (unsigned)rows);
  const size_t size = dtype == DT_F32 ? 4 : 2;
  const bool vec = vocab % 4 == 0 && row_stride % 4 == 0 && reinterpret_cast<uintptr_t>(logits) % (4 * size) == 0 &&
                   reinterpret_cast<uintptr_t>(out) % 16 == 0;
  cudaError_t e = dtype == DT_F32   ? adjust_launch<float>(vec, grid, st, a)
                  : dtype == DT_F16 ? adjust_launch<__half>(vec, grid, st, a)
                                    : adjust_launch<__nv_bfloat16>(vec, grid, st, a);
  if (e == cudaSuccess) e = launch_pdl(pick_kernel, dim3((unsigned)rows), dim3(32), 0, st, a);
  return launched(e, "gsq_adjust_logits");
}

int gsq_record_tokens(const int32_t* tokens, int64_t row_stride, int64_t rows, int64_t n, int64_t vocab, int32_t* seen,
                      int32_t* counts, int generated, gsq_stream_t stream) {
  if (rows < 0 || rows > 65535 || n < 0 || n > (1ll << 30) || vocab <= 0 || vocab > (1ll << 30) || row_stride < 0)
    return fail(GSQ_ERR_SIZE, "gsq_record_tokens: bad shape");
  if (rows == 0 || n == 0) return GSQ_OK;
  if (!tokens || !seen || !counts) return fail(GSQ_ERR_ARG, "gsq_record_tokens: null pointer");
  const int64_t blocks = (rows * n + 255) / 256;
  return launched(launch_pdl(record_kernel, dim3((unsigned)(blocks < 148 * 8 ? blocks : 148 * 8)), dim3(256), 0,
                             (cudaStream_t)stream, tokens, row_stride, rows, n, vocab, (vocab + 31) / 32, seen, counts,
                             generated),
                  "gsq_record_tokens");
}

}  // extern "C"
