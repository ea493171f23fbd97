// Quantised key/value cache: vectors are quantised as they are written
// (gsq_kv_append) and can be read back (gsq_kv_read).
//
// One vector x of one token and head, with m = 127 (int8) or 448 (e4m3):
//   scale = max|x| * (1/m),   code = round to nearest even of x / scale,
// each an IEEE fp32 operation, so that the codes are a function of the inputs
// alone, on any machine.
// A vector that holds Inf or NaN gets the scale NaN and zero codes: it reads
// back as NaN, and attention over it gives NaN, in the rows that see it only.
//
// Bound: HBM bytes (input + D + 4 a vector), or the launch for one token.
// One warp per vector: the whole vector sits in the warp's registers (D / 32
// values a lane), so the maximum is five shuffles and nothing is read twice.
#include <cuda_fp8.h>

#include <cstdio>

#include "gsq_common.cuh"
#include "gsq_host.h"
#include "gsq_kv.h"
#include "../../include/gsq_model.h"

using namespace gsq;

namespace {

constexpr int KV_WARPS = 4;

struct KvArgs {
  const void* src[2];     // k, v (append)
  int64_t sb[2], st[2], sh[2];  // their strides in elements (batch, token, head)
  void* dst[2];           // k, v (read), contiguous [batch, tokens, heads, dim]
  uint8_t* codes[2];      // [batch, heads, cap, dim]
  float* scale[2];        // [batch, heads, cap]
  const int32_t* start;   // first position of sequence b: start[b * start_stride]
  int64_t start_stride;
  const int32_t* counts;  // tokens of sequence b (null: all)
  int64_t tokens, heads, cap, vectors;
  int* err;
};

// Position of vector (b, t) in the cache, or -1: past the sequence's count, or outside the cache.
__device__ __forceinline__ int64_t kv_position(const KvArgs& a, int64_t b, int64_t t, bool* outside) {
  *outside = false;
  if (a.counts && t >= a.counts[b]) return -1;
  const int64_t p = (int64_t)a.start[b * a.start_stride] + t;
  if (p >= 0 && p < a.cap) return p;
  *outside = true;
  return -1;
}

// N consecutive values of T at p, as one or two vector loads where VEC (p 16-byte aligned, or 8-byte for 8 bytes).
template <typename T, int N, bool VEC>
__device__ __forceinline__ void load_n(const T* p, float (&f)[N]) {
  if constexpr (VEC) {
    constexpr int B = sizeof(T) * N;
    static_assert(B == 8 || B % 16 == 0, "whole vector loads");
    alignas(16) T e[N];
    if constexpr (B == 8) {
      *reinterpret_cast<uint2*>(e) = *reinterpret_cast<const uint2*>(p);
    } else {
#pragma unroll
      for (int i = 0; i < B / 16; i++) reinterpret_cast<uint4*>(e)[i] = reinterpret_cast<const uint4*>(p)[i];
    }
#pragma unroll
    for (int i = 0; i < N; i++) f[i] = to_f32(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) f[i] = to_f32(p[i]);
  }
}

// Codes and scale of the warp's vector, N values a lane.
template <int FMT, int N>
__device__ __forceinline__ void quantise(const float (&f)[N], uint8_t (&code)[N], float& scale) {
  float m = 0.f;
  bool finite = true;
#pragma unroll
  for (int i = 0; i < N; i++) {
    m = fmaxf(m, fabsf(f[i]));
    finite = finite && isfinite(f[i]);
  }
  finite = __all_sync(0xffffffffu, finite);
#pragma unroll
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  constexpr float M = FMT == KV_INT8 ? 127.f : 448.f;
  scale = __fmul_rn(m, 1.f / M);
  if (m > 1e38f) scale = fminf(scale, __fdiv_rd(3.402823466e38f, M));  // M * scale stays finite
  if (!finite) scale = __int_as_float(0x7fffffff);
#pragma unroll
  for (int i = 0; i < N; i++) {
    const float y = scale > 0.f ? __fdiv_rn(f[i], scale) : 0.f;  // scale 0 (a zero vector) and NaN: code 0
    if constexpr (FMT == KV_INT8) {
      // a subnormal scale is coarse enough for a quotient past 127
      code[i] = (uint8_t)(int8_t)(int)rintf(fminf(fmaxf(y, -127.f), 127.f));
    } else {
      code[i] = __nv_cvt_float_to_fp8(y, __NV_SATFINITE, __NV_E4M3);
    }
  }
}

template <int N>
__device__ __forceinline__ void store_codes(uint8_t* p, const uint8_t (&c)[N]) {
  uint32_t w[N / 4];
#pragma unroll
  for (int i = 0; i < N / 4; i++)
    w[i] = (uint32_t)c[4 * i] | (uint32_t)c[4 * i + 1] << 8 | (uint32_t)c[4 * i + 2] << 16 | (uint32_t)c[4 * i + 3] << 24;
  if constexpr (N == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  else *reinterpret_cast<uint32_t*>(p) = w[0];
}

template <typename T, int FMT, int D, bool VEC>
__global__ void __launch_bounds__(32 * KV_WARPS) kv_append_kernel(const KvArgs a) {
  constexpr int N = D / 32;
  pdl_launch_dependents();
  pdl_wait();
  const int64_t u = (int64_t)blockIdx.x * KV_WARPS + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (u >= a.vectors) return;
  const int which = blockIdx.y;
  const int64_t h = u % a.heads, t = u / a.heads % a.tokens, b = u / (a.heads * a.tokens);
  bool outside;
  const int64_t p = kv_position(a, b, t, &outside);
  if (p < 0) {
    if (outside && lane == 0 && a.err) atomicExch(a.err, DEV_CACHE_POSITION);
    return;
  }
  float f[N];
  load_n<T, N, VEC>(static_cast<const T*>(a.src[which]) + b * a.sb[which] + t * a.st[which] + h * a.sh[which] + lane * N,
                    f);
  uint8_t code[N];
  float scale;
  quantise<FMT, N>(f, code, scale);
  const int64_t row = (b * a.heads + h) * a.cap + p;
  store_codes<N>(a.codes[which] + row * D + lane * N, code);
  if (lane == 0) a.scale[which][row] = scale;
}

template <int FMT>
__device__ __forceinline__ float code_value(uint8_t c) {
  if constexpr (FMT == KV_INT8) return (float)(int8_t)c;
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3)));
}

// Positions outside the cache, and past a sequence's count, read as zeros.
template <typename T, int FMT, int D>
__global__ void __launch_bounds__(32 * KV_WARPS) kv_read_kernel(const KvArgs a) {
  constexpr int N = D / 32;
  pdl_launch_dependents();
  pdl_wait();
  const int64_t u = (int64_t)blockIdx.x * KV_WARPS + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (u >= a.vectors) return;
  const int which = blockIdx.y;
  const int64_t h = u % a.heads, t = u / a.heads % a.tokens, b = u / (a.heads * a.tokens);
  bool outside;
  const int64_t p = kv_position(a, b, t, &outside);
  alignas(16) T e[N];
#pragma unroll
  for (int i = 0; i < N; i++) e[i] = T(0.f);
  if (p >= 0) {
    const int64_t row = (b * a.heads + h) * a.cap + p;
    const float scale = a.scale[which][row];
    alignas(8) uint8_t c[N];
    const uint8_t* src = a.codes[which] + row * D + lane * N;
    if constexpr (N == 8) *reinterpret_cast<uint2*>(c) = *reinterpret_cast<const uint2*>(src);
    else *reinterpret_cast<uint32_t*>(c) = *reinterpret_cast<const uint32_t*>(src);
#pragma unroll
    for (int i = 0; i < N; i++) store_out(e, sizeof(T) == 4 ? DT_F32 : std::is_same<T, __half>::value ? DT_F16 : DT_BF16, i,
                                          code_value<FMT>(c[i]) * scale);
  }
  T* dst = static_cast<T*>(a.dst[which]) + u * D + lane * N;
  constexpr int B = sizeof(T) * N;
  if constexpr (B == 8) *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(e);
  else
#pragma unroll
    for (int i = 0; i < B / 16; i++) reinterpret_cast<uint4*>(dst)[i] = reinterpret_cast<const uint4*>(e)[i];
}

int fail(int code, const char* msg) { return set_last_error(code, msg); }

int launched(cudaError_t rc, const char* what) {
  if (rc == cudaSuccess) rc = cudaGetLastError();
  if (rc == cudaSuccess) return GSQ_OK;
  char buf[256];
  snprintf(buf, sizeof(buf), "%s: %s", what, cudaGetErrorString(rc));
  return fail(GSQ_ERR_CUDA, buf);
}

template <int FMT, int D>
cudaError_t append_launch(int dtype, bool vec, dim3 grid, cudaStream_t st, const KvArgs& a) {
  const dim3 block(32 * KV_WARPS);
  switch (dtype) {
    case DT_F32:
      return vec ? launch_pdl(kv_append_kernel<float, FMT, D, true>, grid, block, 0, st, a)
                 : launch_pdl(kv_append_kernel<float, FMT, D, false>, grid, block, 0, st, a);
    case DT_F16:
      return vec ? launch_pdl(kv_append_kernel<__half, FMT, D, true>, grid, block, 0, st, a)
                 : launch_pdl(kv_append_kernel<__half, FMT, D, false>, grid, block, 0, st, a);
    default:
      return vec ? launch_pdl(kv_append_kernel<__nv_bfloat16, FMT, D, true>, grid, block, 0, st, a)
                 : launch_pdl(kv_append_kernel<__nv_bfloat16, FMT, D, false>, grid, block, 0, st, a);
  }
}

template <int FMT, int D>
cudaError_t read_launch(int dtype, dim3 grid, cudaStream_t st, const KvArgs& a) {
  const dim3 block(32 * KV_WARPS);
  switch (dtype) {
    case DT_F32: return launch_pdl(kv_read_kernel<float, FMT, D>, grid, block, 0, st, a);
    case DT_F16: return launch_pdl(kv_read_kernel<__half, FMT, D>, grid, block, 0, st, a);
    default: return launch_pdl(kv_read_kernel<__nv_bfloat16, FMT, D>, grid, block, 0, st, a);
  }
}

bool al16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace

namespace gsq {

int kv_check(const char* who, int fmt, const void* kc, const void* vc, const void* ks, const void* vs, int64_t batch,
             int64_t heads, int64_t dim, int64_t cap) {
  char buf[192];
  const char* what = nullptr;
  int code = GSQ_ERR_SIZE;
  if (fmt != KV_INT8 && fmt != KV_FP8) what = "unknown cache format", code = GSQ_ERR_ARG;
  else if (!kc || !vc || !ks || !vs) what = "null cache pointer", code = GSQ_ERR_ARG;
  else if (dim != 128 && dim != 256) what = "head width must be 128 or 256";
  else if (batch < 0 || batch > 65535 || heads <= 0 || heads > 65535) what = "bad batch or head count";
  else if (cap <= 0 || cap > (1ll << 30)) what = "bad cache length";
  else if (!al16(kc) || !al16(vc)) what = "cache codes not 16-byte aligned", code = GSQ_ERR_ALIGN;
  else if (reinterpret_cast<uintptr_t>(ks) % 4 || reinterpret_cast<uintptr_t>(vs) % 4)
    what = "cache scales not 4-byte aligned", code = GSQ_ERR_ALIGN;
  if (!what) return GSQ_OK;
  snprintf(buf, sizeof(buf), "%s: %s", who, what);
  return set_last_error(code, buf);
}

}  // namespace gsq

extern "C" {

int gsq_kv_append(const void* k, const void* v, int dtype, int64_t batch, int64_t tokens, int64_t heads, int64_t dim,
                  const int64_t* k_strides, const int64_t* v_strides, const int32_t* start, int64_t start_stride,
                  const int32_t* counts, int fmt, void* k_codes, void* v_codes, float* k_scale, float* v_scale,
                  int64_t cap, gsq_stream_t stream) {
  int rc = kv_check("gsq_kv_append", fmt, k_codes, v_codes, k_scale, v_scale, batch, heads, dim, cap);
  if (rc) return rc;
  if (dtype != DT_F32 && dtype != DT_F16 && dtype != DT_BF16) return fail(GSQ_ERR_ARG, "gsq_kv_append: bad dtype");
  if (tokens < 0 || tokens > (1ll << 30)) return fail(GSQ_ERR_SIZE, "gsq_kv_append: bad token count");
  if (batch == 0 || tokens == 0) return GSQ_OK;
  if (!k || !v || !start || !k_strides || !v_strides) return fail(GSQ_ERR_ARG, "gsq_kv_append: null pointer");
  const int64_t size = dtype == DT_F32 ? 4 : 2;
  KvArgs a = {};
  a.src[0] = k;
  a.src[1] = v;
  // vector loads where every vector starts on a 16-byte boundary (two-byte values of 128-wide heads: 8 bytes a lane)
  bool vec = al16(k) && al16(v);
  for (int i = 0; i < 2; i++) {
    const int64_t* s = i ? v_strides : k_strides;
    a.sb[i] = s[0];
    a.st[i] = s[1];
    a.sh[i] = s[2];
    for (int j = 0; j < 3; j++) vec = vec && s[j] * size % 16 == 0;
    if (reinterpret_cast<uintptr_t>(a.src[i]) % size) return fail(GSQ_ERR_ALIGN, "gsq_kv_append: unaligned input");
  }
  a.codes[0] = static_cast<uint8_t*>(k_codes);
  a.codes[1] = static_cast<uint8_t*>(v_codes);
  a.scale[0] = k_scale;
  a.scale[1] = v_scale;
  a.start = start;
  a.start_stride = start_stride;
  a.counts = counts;
  a.tokens = tokens;
  a.heads = heads;
  a.cap = cap;
  a.vectors = batch * tokens * heads;
  a.err = device_error_word();
  if ((a.vectors + KV_WARPS - 1) / KV_WARPS > INT32_MAX) return fail(GSQ_ERR_SIZE, "gsq_kv_append: too many vectors");
  const dim3 grid((unsigned)((a.vectors + KV_WARPS - 1) / KV_WARPS), 2);
  cudaStream_t st = (cudaStream_t)stream;
  const cudaError_t e = fmt == KV_INT8 ? (dim == 256 ? append_launch<KV_INT8, 256>(dtype, vec, grid, st, a)
                                                     : append_launch<KV_INT8, 128>(dtype, vec, grid, st, a))
                                       : (dim == 256 ? append_launch<KV_FP8, 256>(dtype, vec, grid, st, a)
                                                     : append_launch<KV_FP8, 128>(dtype, vec, grid, st, a));
  return launched(e, "gsq_kv_append");
}

int gsq_kv_read(int fmt, const void* k_codes, const void* v_codes, const float* k_scale, const float* v_scale,
                int64_t batch, int64_t heads, int64_t cap, int64_t dim, const int32_t* start, int64_t start_stride,
                const int32_t* counts, int64_t tokens, void* k, void* v, int dtype, gsq_stream_t stream) {
  int rc = kv_check("gsq_kv_read", fmt, k_codes, v_codes, k_scale, v_scale, batch, heads, dim, cap);
  if (rc) return rc;
  if (dtype != DT_F32 && dtype != DT_F16 && dtype != DT_BF16) return fail(GSQ_ERR_ARG, "gsq_kv_read: bad dtype");
  if (tokens < 0 || tokens > (1ll << 30)) return fail(GSQ_ERR_SIZE, "gsq_kv_read: bad token count");
  if (batch == 0 || tokens == 0) return GSQ_OK;
  if (!k || !v || !start) return fail(GSQ_ERR_ARG, "gsq_kv_read: null pointer");
  if (!al16(k) || !al16(v)) return fail(GSQ_ERR_ALIGN, "gsq_kv_read: outputs not 16-byte aligned");
  KvArgs a = {};
  a.dst[0] = k;
  a.dst[1] = v;
  a.codes[0] = static_cast<uint8_t*>(const_cast<void*>(k_codes));
  a.codes[1] = static_cast<uint8_t*>(const_cast<void*>(v_codes));
  a.scale[0] = const_cast<float*>(k_scale);
  a.scale[1] = const_cast<float*>(v_scale);
  a.start = start;
  a.start_stride = start_stride;
  a.counts = counts;
  a.tokens = tokens;
  a.heads = heads;
  a.cap = cap;
  a.vectors = batch * tokens * heads;
  if ((a.vectors + KV_WARPS - 1) / KV_WARPS > INT32_MAX) return fail(GSQ_ERR_SIZE, "gsq_kv_read: too many vectors");
  const dim3 grid((unsigned)((a.vectors + KV_WARPS - 1) / KV_WARPS), 2);
  cudaStream_t st = (cudaStream_t)stream;
  const cudaError_t e = fmt == KV_INT8 ? (dim == 256 ? read_launch<KV_INT8, 256>(dtype, grid, st, a)
                                                     : read_launch<KV_INT8, 128>(dtype, grid, st, a))
                                       : (dim == 256 ? read_launch<KV_FP8, 256>(dtype, grid, st, a)
                                                     : read_launch<KV_FP8, 128>(dtype, grid, st, a));
  return launched(e, "gsq_kv_read");
}

}  // extern "C"
