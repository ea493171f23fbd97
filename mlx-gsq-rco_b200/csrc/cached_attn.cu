// Attention of the newest tokens of each sequence over the quantised cache
// (gsq_cached_attention): one warp per query row, an online softmax over the
// positions the row sees.
#include <atomic>
#include <cstdio>

#include "attn_token.cuh"
#include "gsq_host.h"
#include "../../include/gsq_model.h"

using namespace gsq;

namespace {

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
  if (r >= (int64_t)a.batch * a.n * a.heads) return;
  const int64_t h = r % a.heads, i = r / a.heads % a.n, b = r / ((int64_t)a.heads * a.n);
  const int64_t kh = h / a.group;
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
bool al(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

template <typename T, int FMT>
cudaError_t simple(int64_t dim, dim3 grid, cudaStream_t st, const AttnArgs& a) {
  return dim == 256 ? launch_pdl(attn_simple_kernel<T, FMT, 256>, grid, dim3(128), 0, st, a)
                    : launch_pdl(attn_simple_kernel<T, FMT, 128>, grid, dim3(128), 0, st, a);
}

constexpr int SMS = 148;

// Which kernel a call takes, over how many CTAs, and its scratch.
struct Plan {
  int nt;           // 8-row tiles of the token kernel (0: the simple kernel)
  int ctas, rows8;
  size_t workspace;
};

Plan plan_of(int64_t batch, int64_t n, int64_t heads, int64_t kv, int64_t dim, int64_t cap) {
  Plan p = {};
  const int64_t rows = n * (heads / kv);
  if (rows > 16) return p;
  p.nt = rows <= 8 ? 1 : 2;
  p.rows8 = 8 * p.nt;
  const int64_t tiles = batch * kv * ((cap + AT_TILE - 1) / AT_TILE);
  p.ctas = (int)(tiles < SMS ? tiles : SMS);
  p.workspace = (size_t)2 * p.ctas * p.rows8 * (dim + 2) * sizeof(float);
  return p;
}

template <typename T, int FMT, int D, int NT>
cudaError_t token_launch(cudaStream_t st, const AttnArgs& a) {
  auto kernel = attn_token_kernel<T, FMT, D, NT>;
  constexpr int smem = AtGeom<D, NT>::SMEM;
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64 || !(done.load(std::memory_order_relaxed) >> dev & 1)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    if (dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  e = launch_pdl(kernel, dim3((unsigned)a.ctas), dim3(32 * AT_WARPS), smem, st, a);
  if (e != cudaSuccess) return e;
  return launch_pdl(attn_join_kernel<T, D, AT_TILE>, dim3((unsigned)(a.batch * a.kv * a.n * a.group)), dim3(256), 0, st, a);
}

template <typename T, int FMT>
cudaError_t token(int nt, cudaStream_t st, const AttnArgs& a) {
  if (a.dim == 256) return nt == 1 ? token_launch<T, FMT, 256, 1>(st, a) : token_launch<T, FMT, 256, 2>(st, a);
  return nt == 1 ? token_launch<T, FMT, 128, 1>(st, a) : token_launch<T, FMT, 128, 2>(st, a);
}

}  // namespace

extern "C" {

size_t gsq_cached_attention_workspace_size(int64_t batch, int64_t n, int64_t heads, int64_t kv_heads, int64_t dim,
                                           int64_t cap) {
  if (batch <= 0 || n <= 0 || heads <= 0 || kv_heads <= 0 || dim <= 0 || cap <= 0) return 0;
  return plan_of(batch, n, heads, kv_heads, dim, cap).workspace;
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
  if (batch * kv_heads * ((cap + AT_TILE - 1) / AT_TILE) > INT32_MAX || batch * n * heads > INT32_MAX)
    return fail(GSQ_ERR_SIZE, "gsq_cached_attention: too much work for one call");
  for (int i = 0; i < 3; i++)
    if (q_strides[i] % 8) return fail(GSQ_ERR_ALIGN, "gsq_cached_attention: rows of q not 16-byte aligned");
  if (!al(q, 16) || !al(out, 16) || !al(gate, 4))
    return fail(GSQ_ERR_ALIGN, "gsq_cached_attention: q or out not 16-byte aligned, or gate not aligned");
  AttnArgs a = {};
  a.q = q;
  a.qb = q_strides[0];
  a.qn = q_strides[1];
  a.qh = q_strides[2];
  a.kc = static_cast<const uint8_t*>(k_codes);
  a.vc = static_cast<const uint8_t*>(v_codes);
  a.ks = k_scale;
  a.vs = v_scale;
  a.batch = (int)batch;
  a.n = (int)n;
  a.heads = (int)heads;
  a.kv = (int)kv_heads;
  a.group = (int)(heads / kv_heads);
  a.dim = (int)dim;
  a.words = (int)((n + 31) / 32);
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
  const Plan plan = plan_of(batch, n, heads, kv_heads, dim, cap);
  if (plan.workspace && (!workspace || workspace_bytes < plan.workspace))
    return fail(GSQ_ERR_WORKSPACE, "gsq_cached_attention: workspace missing or too small");
  if (!al(workspace, 256)) return fail(GSQ_ERR_ALIGN, "gsq_cached_attention: workspace not 256-byte aligned");
  a.ctas = plan.ctas;
  a.rows8 = plan.rows8;
  a.part = static_cast<float*>(workspace);
  a.stat = a.part + (size_t)2 * a.ctas * a.rows8 * dim;
  cudaError_t e;
  if (plan.nt) {
    e = dtype == DT_F16 ? (fmt == KV_INT8 ? token<__half, KV_INT8>(plan.nt, st, a) : token<__half, KV_FP8>(plan.nt, st, a))
                        : (fmt == KV_INT8 ? token<__nv_bfloat16, KV_INT8>(plan.nt, st, a)
                                          : token<__nv_bfloat16, KV_FP8>(plan.nt, st, a));
  } else {
    const dim3 grid((unsigned)((batch * n * heads + 3) / 4));
    e = dtype == DT_F16 ? (fmt == KV_INT8 ? simple<__half, KV_INT8>(dim, grid, st, a) : simple<__half, KV_FP8>(dim, grid, st, a))
                        : (fmt == KV_INT8 ? simple<__nv_bfloat16, KV_INT8>(dim, grid, st, a) : simple<__nv_bfloat16, KV_FP8>(dim, grid, st, a));
  }
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e == cudaSuccess) return GSQ_OK;
  char buf[256];
  snprintf(buf, sizeof(buf), "gsq_cached_attention: %s", cudaGetErrorString(e));
  return fail(GSQ_ERR_CUDA, buf);
}

}  // extern "C"
