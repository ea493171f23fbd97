// Attention of the newest tokens of each sequence over the quantised cache
// (gsq_cached_attention): which kernel, its launches and checks.  The kernels
// are in attn_token.cuh (few rows per key/value head: the cache's bytes bound
// it) and attn_rows.cuh (many rows: the tensor core).
#include <algorithm>
#include <atomic>
#include <cstdio>

#include "attn_rows.cuh"
#include "attn_token.cuh"
#include "gsq_host.h"
#include "../../include/gsq_model.h"

using namespace gsq;

namespace {

int fail(int code, const char* msg) { return set_last_error(code, msg); }
bool al(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

constexpr int SMS = 148;

// Which kernel a call takes, over how many CTAs, and its scratch.
struct Plan {
  int nt;           // 8-row tiles of the token kernel; 0: the row-block kernel
  int cluster;      // token kernel by units: CTAs of a unit; 0: tiles split evenly
  int blocks;       // and its units per key/value head
  int joins;        // row-block kernel: CTAs that join one unit's parts
  int ctas, rows8;
  int64_t tiles;    // at most, over all sequences at full length
  size_t workspace;
};

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Token kernel by units of up to 16 rows: as many CTAs for each unit, up to 8, as fill `most` slots; twice as many where
// a CTA would still have more than 64 tiles, since units of unlike length then even out (64 sequences, 4 heads of 256:
// up to 8000 positions 154 us and with twice as many CTAs 101, all of 8000 169 and 175; up to 2304 positions, 36 tiles,
// 49 and 42, but all of 2304 54 and 63; of an earlier state of the kernel, to be compared with each other).
void plan_units(Plan& p, int64_t units, int64_t most, int64_t tiles) {
  p.cluster = 1;
  while (p.cluster < 8 && units * p.cluster * (tiles > 64 * p.cluster ? 1 : 2) <= most) p.cluster *= 2;
  p.ctas = (int)(units * p.cluster);
}

// Up to 16 rows per key/value head the token kernel reads the cache once at the memory's rate; its tensor-core tiles
// and registers hold two groups of eight rows.  By units up to 8192 positions: 64 ragged sequences of up to 2304 take
// 53 us and one takes 14, against 67 and 17 with the tiles split evenly and joined by a second launch.  Units of longer
// caches may differ by more than the CTA slots even out, and few units of one need more than 8 CTAs each.
//
// More rows: the row-block kernel; or, of caches up to 8192 positions, several units of 16 rows for the token kernel,
// which read the cache again (from L2).  A tile of 64 positions takes a CTA about as long in either, 1.0 us at 128
// dimensions and 1.7 at 256.  In these terms a wave of the token kernel's CTAs costs 5 and its tiles; the row-block
// kernel 8, 1 for every 32 rows (queries loaded, results stored), its tiles, and the joining launch 1 for every 1200
// rows of parts.  Fitted to measurements with 4 heads of 256, such as (us, token kernel and row blocks): one sequence,
// 40 rows, 2000 positions 18 and 20; 128 rows, 700 positions 16 and 24; 24 rows, 8000 positions 32 and 25; 8 sequences
// of 2000 positions, 24 rows 26 and 34, 96 rows 64 and 44.  Past 256 rows the row blocks are full.
Plan plan_of(int64_t batch, int64_t n, int64_t heads, int64_t kv, int64_t dim, int64_t cap) {
  Plan p = {};
  const int64_t rows = n * (heads / kv), cached = batch * kv;  // heads in the cache
  p.blocks = 1;
  if (rows > 16) {
    const int64_t units = cached * ceil_div(rows, AR_M), tiles = ceil_div(cap, AR_TILE);
    p.rows8 = AR_M;
    p.tiles = units * tiles;
    p.ctas = (int)std::min<int64_t>(p.tiles, SMS);
    p.joins = units <= 8 ? 32 : 16;  // few units are in many parts each: 1 unit of 125, 128 rows 42 us with 32, 52 with 16
    if (rows <= 256 && cap <= 8192) {
      Plan t = {};
      t.nt = 2;
      t.rows8 = 16;
      t.blocks = (int)ceil_div(rows, 16);
      t.tiles = cached * t.blocks * tiles;
      plan_units(t, cached * t.blocks, SMS * 2, tiles);
      const int64_t full = std::min<int64_t>(rows, AR_M), parts = ceil_div(p.ctas, units);
      if (ceil_div(t.ctas, SMS * 2) * (5 + ceil_div(tiles, t.cluster)) <=
          8 + full / 32 + ceil_div(p.tiles, p.ctas) + (parts > 1 ? parts * full / 1200 : 0))
        return t;
    }
  } else {
    p.nt = rows <= 8 ? 1 : 2;
    p.rows8 = 8 * p.nt;
    p.tiles = cached * ceil_div(cap, AT_TILE);
    const int64_t most = SMS * (dim == 128 && p.nt == 1 ? 3 : 2);  // CTAs that run at once
    if (cap <= 8192) {
      plan_units(p, cached, most, ceil_div(cap, AT_TILE));
      return p;
    }
    p.ctas = (int)std::min<int64_t>(p.tiles, most);
  }
  p.workspace = (size_t)2 * p.ctas * p.rows8 * (dim + 2) * sizeof(float) + p.ctas * sizeof(Joint);
  return p;
}

// Opts `kernel` in to its dynamic shared memory, once per device (`done`: one bit each).
template <typename K>
cudaError_t allow_smem(K kernel, int bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || (dev < 64 && done.load(std::memory_order_relaxed) >> dev & 1)) return e;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
  return e;
}

template <typename T, int FMT, int D, int NT, bool UNITS>
cudaError_t token_launch(cudaStream_t st, const AttnArgs& a) {
  static std::atomic<uint64_t> done{0};
  constexpr int smem = AtGeom<D, NT>::SMEM;
  auto kernel = attn_token_kernel<T, FMT, D, NT, UNITS>;
  cudaError_t e = allow_smem(kernel, smem, done);
  if (e != cudaSuccess) return e;
  const dim3 grid((unsigned)a.ctas), block(32 * AT_WARPS);
  if (UNITS && a.cluster > 1) return launch_pdl_cluster(kernel, grid, block, a.cluster, st, smem, a);
  e = launch_pdl(kernel, grid, block, smem, st, a);
  if (e != cudaSuccess || UNITS) return e;
  return launch_pdl(attn_join_kernel<T, D, AtShape>, dim3((unsigned)a.ctas, (unsigned)(a.n * a.group)), dim3(256), 0, st,
                    a);
}

template <typename T, int FMT, int D>
cudaError_t rows_launch(cudaStream_t st, const AttnArgs& a) {
  static std::atomic<uint64_t> done{0};
  constexpr int smem = ArGeom<D>::SMEM;
  cudaError_t e = allow_smem(attn_rows_kernel<T, FMT, D>, smem, done);
  if (e == cudaSuccess)
    e = launch_pdl(attn_rows_kernel<T, FMT, D>, dim3((unsigned)a.ctas), dim3(AR_THREADS), smem, st, a);
  if (e != cudaSuccess) return e;
  return launch_pdl(attn_join_kernel<T, D, ArShape>, dim3((unsigned)a.ctas, a.joins), dim3(256), 0, st, a);
}

template <typename T, int FMT, int D>
cudaError_t attend(const Plan& p, cudaStream_t st, const AttnArgs& a) {
  if (p.nt == 0) return rows_launch<T, FMT, D>(st, a);
  if (p.nt == 1) return p.cluster ? token_launch<T, FMT, D, 1, true>(st, a) : token_launch<T, FMT, D, 1, false>(st, a);
  return p.cluster ? token_launch<T, FMT, D, 2, true>(st, a) : token_launch<T, FMT, D, 2, false>(st, a);
}

template <typename T>
cudaError_t attend(int fmt, const Plan& p, cudaStream_t st, const AttnArgs& a) {
  if (fmt == KV_INT8) return a.dim == 256 ? attend<T, KV_INT8, 256>(p, st, a) : attend<T, KV_INT8, 128>(p, st, a);
  return a.dim == 256 ? attend<T, KV_FP8, 256>(p, st, a) : attend<T, KV_FP8, 128>(p, st, a);
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
  const Plan plan = plan_of(batch, n, heads, kv_heads, dim, cap);
  if (plan.tiles > INT32_MAX || batch * n * heads > INT32_MAX)
    return fail(GSQ_ERR_SIZE, "gsq_cached_attention: too much work for one call");
  for (int i = 0; i < 3; i++)
    if (q_strides[i] % 8) return fail(GSQ_ERR_ALIGN, "gsq_cached_attention: rows of q not 16-byte aligned");
  if (!al(q, 16) || !al(out, 16) || !words_aligned({start, counts, tree, gate}))
    return fail(GSQ_ERR_ALIGN, "gsq_cached_attention: q or out not 16-byte aligned, or 4-byte values not aligned");
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
  if (plan.workspace && (!workspace || workspace_bytes < plan.workspace))
    return fail(GSQ_ERR_WORKSPACE, "gsq_cached_attention: workspace missing or too small");
  if (!al(workspace, 256)) return fail(GSQ_ERR_ALIGN, "gsq_cached_attention: workspace not 256-byte aligned");
  a.ctas = plan.ctas;
  a.rows8 = plan.rows8;
  a.part = static_cast<float*>(workspace);
  a.stat = a.part + (size_t)2 * a.ctas * a.rows8 * dim;
  a.joints = reinterpret_cast<Joint*>(a.stat + (size_t)2 * a.ctas * a.rows8 * 2);
  a.cluster = plan.cluster;
  a.blocks = plan.blocks;
  a.joins = plan.joins;
  a.err = device_error_word();
  cudaError_t e = dtype == DT_F16 ? attend<__half>(fmt, plan, st, a) : attend<__nv_bfloat16>(fmt, plan, st, a);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e == cudaSuccess) return GSQ_OK;
  char buf[256];
  snprintf(buf, sizeof(buf), "gsq_cached_attention: %s", cudaGetErrorString(e));
  return fail(GSQ_ERR_CUDA, buf);
}

}  // extern "C"
