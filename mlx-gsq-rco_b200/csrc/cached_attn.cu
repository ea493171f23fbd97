// Attention of the newest tokens of each sequence over the quantised cache
// (gsq_cached_attention): one warp per query row, an online softmax over the
// positions the row sees.
#include <cuda_fp8.h>

#include <cstdio>

#include "gsq_common.cuh"
#include "gsq_host.h"
#include "gsq_kv.h"
#include "../../include/gsq_model.h"

using namespace gsq;

namespace {

struct AttnArgs {
  const void* q;
  int64_t qb, qn, qh;  // strides in elements (sequence, token, head)
  const uint8_t *kc, *vc;
  const float *ks, *vs;
  int64_t batch, n, heads, kv, cap;
  const int32_t* start;
  int64_t start_stride;
  const int32_t* counts;
  const int32_t* tree;
  int64_t tree_stride;
  const float* gate;
  int64_t gb, gn, gh;
  float scale;
  void* out;
};

template <int FMT>
__device__ __forceinline__ float code_value(uint8_t c) {
  if constexpr (FMT == KV_INT8) return (float)(int8_t)c;
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3)));
}

template <typename T, int FMT, int D>
__global__ void __launch_bounds__(128) attn_simple_kernel(const AttnArgs a) {
  constexpr int N = D / 32;
  pdl_launch_dependents();
  pdl_wait();
  const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (r >= a.batch * a.n * a.heads) return;
  const int64_t h = r % a.heads, i = r / a.heads % a.n, b = r / (a.heads * a.n);
  const int64_t kh = h / (a.heads / a.kv);
  T* out = static_cast<T*>(a.out) + r * D + lane * N;
  const int64_t base = a.start[b * a.start_stride];
  const int64_t count = a.counts ? a.counts[b] : a.n;
  float q[N], o[N];
  const T* qp = static_cast<const T*>(a.q) + b * a.qb + i * a.qn + h * a.qh + lane * N;
#pragma unroll
  for (int e = 0; e < N; e++) {
    q[e] = to_f32(qp[e]);
    o[e] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  int64_t end = a.tree ? base + count : base + i + 1;
  if (end > a.cap) end = a.cap;
  if (i >= count) end = 0;
  const int32_t* bits = a.tree ? a.tree + b * a.tree_stride + i * ((a.n + 31) / 32) : nullptr;
  const int64_t row0 = (b * a.kv + kh) * a.cap;
  for (int64_t p = 0; p < end; p++) {
    if (bits && p >= base && !((uint32_t)bits[(p - base) >> 5] >> ((p - base) & 31) & 1)) continue;
    const uint8_t* kp = a.kc + (row0 + p) * D + lane * N;
    const uint8_t* vp = a.vc + (row0 + p) * D + lane * N;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < N; e++) s = fmaf(q[e], code_value<FMT>(kp[e]), s);
#pragma unroll
    for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    s *= a.ks[row0 + p] * a.scale;
    const float mn = fmaxf(m, s), c = m == -INFINITY ? 0.f : __expf(m - mn), w = __expf(s - mn);
    l = l * c + w;
#pragma unroll
    for (int e = 0; e < N; e++) o[e] = o[e] * c + w * a.vs[row0 + p] * code_value<FMT>(vp[e]);
    m = mn;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const float* g = a.gate ? a.gate + b * a.gb + i * a.gn + h * a.gh + lane * N : nullptr;
#pragma unroll
  for (int e = 0; e < N; e++) {
    float y = o[e] * inv;
    if (g) y /= 1.f + __expf(-g[e]);
    store_out(out, std::is_same<T, __half>::value ? DT_F16 : DT_BF16, e, y);
  }
}

int fail(int code, const char* msg) { return set_last_error(code, msg); }

template <typename T, int FMT>
cudaError_t simple(int64_t dim, dim3 grid, cudaStream_t st, const AttnArgs& a) {
  return dim == 256 ? launch_pdl(attn_simple_kernel<T, FMT, 256>, grid, dim3(128), 0, st, a)
                    : launch_pdl(attn_simple_kernel<T, FMT, 128>, grid, dim3(128), 0, st, a);
}

}  // namespace

extern "C" {

size_t gsq_cached_attention_workspace_size(int64_t batch, int64_t n, int64_t heads, int64_t kv_heads, int64_t dim,
                                           int64_t cap) {
  return 0;
}

int gsq_cached_attention(const void* q, int dtype, const int64_t* q_strides, int64_t batch, int64_t n, int64_t heads,
                         int64_t kv_heads, int64_t dim, int fmt, const void* k_codes, const void* v_codes,
                         const float* k_scale, const float* v_scale, int64_t cap, const int32_t* start,
                         int64_t start_stride, const int32_t* counts, const int32_t* tree, int64_t tree_stride,
                         const float* gate, const int64_t* gate_strides, float scale, void* out, void* workspace,
                         size_t workspace_bytes, gsq_stream_t stream) {
  int rc = kv_check("gsq_cached_attention", fmt, k_codes, v_codes, k_scale, v_scale, batch, kv_heads, dim, cap);
  if (rc) return rc;
  if (dtype != DT_F16 && dtype != DT_BF16) return fail(GSQ_ERR_ARG, "gsq_cached_attention: queries must be fp16 or bf16");
  if (heads <= 0 || heads % kv_heads || heads > 65535)
    return fail(GSQ_ERR_SIZE, "gsq_cached_attention: the query heads must be a multiple of the key/value heads");
  if (n < 0 || n > 65536 || (tree && n > 1024)) return fail(GSQ_ERR_SIZE, "gsq_cached_attention: too many new tokens");
  if (batch == 0 || n == 0) return GSQ_OK;
  if (!q || !q_strides || !start || !out || (gate && !gate_strides))
    return fail(GSQ_ERR_ARG, "gsq_cached_attention: null pointer");
  AttnArgs a = {};
  a.q = q;
  a.qb = q_strides[0];
  a.qn = q_strides[1];
  a.qh = q_strides[2];
  a.kc = static_cast<const uint8_t*>(k_codes);
  a.vc = static_cast<const uint8_t*>(v_codes);
  a.ks = k_scale;
  a.vs = v_scale;
  a.batch = batch;
  a.n = n;
  a.heads = heads;
  a.kv = kv_heads;
  a.cap = cap;
  a.start = start;
  a.start_stride = start_stride;
  a.counts = counts;
  a.tree = tree;
  a.tree_stride = tree_stride;
  a.gate = gate;
  if (gate) {
    a.gb = gate_strides[0];
    a.gn = gate_strides[1];
    a.gh = gate_strides[2];
  }
  a.scale = scale;
  a.out = out;
  cudaStream_t st = (cudaStream_t)stream;
  const dim3 grid((unsigned)((batch * n * heads + 3) / 4));
  cudaError_t e = dtype == DT_F16 ? (fmt == KV_INT8 ? simple<__half, KV_INT8>(dim, grid, st, a) : simple<__half, KV_FP8>(dim, grid, st, a))
                                  : (fmt == KV_INT8 ? simple<__nv_bfloat16, KV_INT8>(dim, grid, st, a) : simple<__nv_bfloat16, KV_FP8>(dim, grid, st, a));
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e == cudaSuccess) return GSQ_OK;
  char buf[256];
  snprintf(buf, sizeof(buf), "gsq_cached_attention: %s", cudaGetErrorString(e));
  return fail(GSQ_ERR_CUDA, buf);
}

}  // extern "C"
