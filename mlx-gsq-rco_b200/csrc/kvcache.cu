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
// Eight values a lane, a vector of 256 in a warp's registers or two of 128, so
// nothing is read twice; a warp takes KV_EACH times as many, all
// loaded before the first is worked on.  Measured with 8 x 1999 tokens of 4
// heads of 256, bf16: append 33 us (98 MB, 3.0 TB/s: instructions, and waits
// for loads), read 15 us of e4m3 (6.5 TB/s: HBM), 18 us of int8.
#include <cuda_fp8.h>

#include <cstdio>

#include "gsq_common.cuh"
#include "gsq_host.h"
#include "gsq_kv.h"
#include "kv_codes.cuh"
#include "../../include/gsq_model.h"

using namespace gsq;

namespace {

constexpr int KV_WARPS = 4;  // per CTA
constexpr int KV_EACH = 4;   // vectors per lane

struct KvArgs {
  const void* src[2];     // k, v (append)
  int64_t sb[2], st[2], sh[2];  // their strides in elements (batch, token, head)
  void* dst[2];           // k, v (read), contiguous [batch, tokens, heads, dim]
  uint8_t* codes[2];      // [batch, heads, cap, dim]
  float* scale[2];        // [batch, heads, cap]
  const int32_t* start;   // first position of sequence b: start[b * start_stride]
  int64_t start_stride;
  const int32_t* counts;  // tokens of sequence b (null: all)
  int tokens, heads;
  int64_t cap;
  int* err;
};

// Sequence b's first position and its tokens (past them: padding).
struct KvSpan {
  int start, count;
};
__device__ __forceinline__ KvSpan kv_span(const KvArgs& a, int b) {
  return {a.start[(int64_t)b * a.start_stride], a.counts ? min(a.counts[b], a.tokens) : a.tokens};
}

// N consecutive values of T at p, as one or two vector loads where VEC (p 16-byte aligned).
template <typename T, int N, bool VEC>
__device__ __forceinline__ void load_n(const T* p, float (&f)[N]) {
  if constexpr (VEC) {
    constexpr int B = sizeof(T) * N;
    static_assert(B % 16 == 0, "whole vector loads");
    alignas(16) T e[N];
#pragma unroll
    for (int i = 0; i < B / 16; i++) reinterpret_cast<uint4*>(e)[i] = reinterpret_cast<const uint4*>(p)[i];
#pragma unroll
    for (int i = 0; i < N; i++) f[i] = to_f32(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) f[i] = to_f32(p[i]);
  }
}

// Codes (one byte each, in order) and scale of the vector that the lanes of `lanes` hold, N values each.
template <int FMT, int N>
__device__ __forceinline__ void quantise(const float (&f)[N], uint32_t (&code)[N / 4], float& scale,
                                         uint32_t lanes = 0xffffffffu) {
  // the largest |x| by its bits, which for Inf and NaN are above every finite number's
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < N; i++) top = max(top, __float_as_uint(f[i]) & 0x7fffffffu);
  top = __reduce_max_sync(lanes, top);
  const float m = __uint_as_float(top);
  constexpr float M = FMT == KV_INT8 ? 127.f : 448.f;
  scale = __fmul_rn(m, 1.f / M);
  if (m > 1e38f) scale = fminf(scale, __fdiv_rd(3.402823466e38f, M));  // M * scale stays finite
  if (top >= 0x7f800000u) scale = __int_as_float(0x7fffffff);
  // The quotient correctly rounded, by Markstein's theorem: with y the correctly rounded reciprocal and q within one
  // unit of x / scale, q + (x - q scale) y rounds to it. q is x times the reciprocal in two parts, neither negative, so
  // that a zero keeps its sign. The remainder is exact as long as q scale does not underflow, which for scales from
  // 2^-60 on only concerns quotients of code 0. (A product with the reciprocal alone, rounded both ways, and a division
  // where the codes differed, took 38 us where this takes 33: 39 % of bf16 vectors hold a tie of int8, such as a value
  // half as large as the largest.)
  if (scale >= 0x1p-60f) {  // the same for the vector's lanes
    const float y = __frcp_rn(scale);
    const float high = __uint_as_float(__float_as_uint(y) - (fmaf(-scale, y, 1.f) < 0.f ? 1u : 0u));
    const float low = fmaf(-scale, high, 1.f) * y;
    const f32x2 high2 = pair(high, high), low2 = pair(low, low), minus2 = pair(-y, -y), scale2 = pair(scale, scale);
    auto quotient = [&](float a, float b) {
      const f32x2 x = pair(a, b), q = fma2(x, high2, mul2(x, low2));
      return fma2(fma2(q, scale2, pair(-a, -b)), minus2, q);
    };
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const f32x2 a = quotient(f[i], f[i + 1]), b = quotient(f[i + 2], f[i + 3]);
      if constexpr (FMT == KV_INT8) {
        const f32x2 R = pair(12582912.f, 12582912.f);  // 1.5 * 2^23: a sum's low bits are the nearest integer, ties to even
        const float2 u = halves(add2(a, R)), v = halves(add2(b, R));
        code[i / 4] = __byte_perm(__byte_perm(__float_as_uint(u.x), __float_as_uint(u.y), 0x0040),
                                  __byte_perm(__float_as_uint(v.x), __float_as_uint(v.y), 0x0040), 0x5410);
      } else {
        const uint32_t u = __nv_cvt_float2_to_fp8x2(halves(a), __NV_SATFINITE, __NV_E4M3);
        code[i / 4] = __byte_perm(u, __nv_cvt_float2_to_fp8x2(halves(b), __NV_SATFINITE, __NV_E4M3), 0x5410);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      uint32_t w = 0;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const float y = scale > 0.f ? __fdiv_rn(f[i + e], scale) : 0.f;  // scale 0 (a zero vector) and NaN: code 0
        uint32_t c;
        if constexpr (FMT == KV_INT8)  // a subnormal scale is coarse enough for a quotient past 127
          c = (uint32_t)(int)rintf(fminf(fmaxf(y, -127.f), 127.f)) & 0xffu;
        else
          c = __nv_cvt_float_to_fp8(y, __NV_SATFINITE, __NV_E4M3);
        w |= c << 8 * e;
      }
      code[i / 4] = w;
    }
  }
}

// Where a lane's vectors of D values lie: vector `first` + i * PER_WARP, token t and head h, values from `at` on.
template <int D>
struct KvLane {
  static constexpr int LANES = D / 8, PER_WARP = 32 / LANES;
  unsigned first;
  int t, h, at;
  uint32_t lanes;  // that share its vectors

  __device__ explicit KvLane(int heads) {
    const int lane = threadIdx.x & 31;
    first = (blockIdx.x * KV_WARPS + (threadIdx.x >> 5)) * (KV_EACH * PER_WARP) + lane / LANES;
    t = first / (unsigned)heads;
    h = first % (unsigned)heads;
    at = lane % LANES * 8;
    lanes = PER_WARP == 1 ? 0xffffffffu : 0xffffu << (lane / LANES * LANES);
  }
  __device__ void next(int heads) {
    h += PER_WARP;
    while (h >= heads) h -= heads, t++;
  }
};

template <typename T, int FMT, int D, bool VEC>
__global__ void __launch_bounds__(32 * KV_WARPS) kv_append_kernel(const KvArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  KvLane<D> lane(a.heads);
  const int which = blockIdx.z, b = blockIdx.y;
  float f[KV_EACH][8];
  int64_t row[KV_EACH];  // of codes and scales, or -1
  const KvSpan span = kv_span(a, b);
  const T* src = static_cast<const T*>(a.src[which]) + b * a.sb[which] + lane.at;
#pragma unroll
  for (int i = 0; i < KV_EACH; i++) {
    row[i] = -1;
    if (lane.t < span.count) {
      const int64_t p = (int64_t)span.start + lane.t;
      if (p >= 0 && p < a.cap) {
        row[i] = ((int64_t)b * a.heads + lane.h) * a.cap + p;
        load_n<T, 8, VEC>(src + lane.t * a.st[which] + lane.h * a.sh[which], f[i]);
      } else if (lane.at == 0 && a.err) {
        atomicExch(a.err, DEV_CACHE_POSITION);
      }
    }
    lane.next(a.heads);
  }
#pragma unroll
  for (int i = 0; i < KV_EACH; i++) {
    if (row[i] < 0) continue;
    uint32_t code[2];
    float scale;
    quantise<FMT, 8>(f[i], code, scale, lane.lanes);
    *reinterpret_cast<uint2*>(a.codes[which] + row[i] * D + lane.at) = make_uint2(code[0], code[1]);
    if (lane.at == 0) a.scale[which][row[i]] = scale;
  }
}

// Positions outside the cache, and past a sequence's count, read as zeros.
template <typename T, int FMT, int D>
__global__ void __launch_bounds__(32 * KV_WARPS) kv_read_kernel(const KvArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  KvLane<D> lane(a.heads);
  const unsigned vectors = a.tokens * a.heads;
  const int which = blockIdx.z, b = blockIdx.y;
  uint32_t c[KV_EACH][2];
  float scale[KV_EACH];
  const KvSpan span = kv_span(a, b);
#pragma unroll
  for (int i = 0; i < KV_EACH; i++) {
    scale[i] = 0.f;
    c[i][0] = c[i][1] = 0u;
    const int64_t p = (int64_t)span.start + lane.t;
    if (lane.t < span.count && p >= 0 && p < a.cap) {
      const int64_t row = ((int64_t)b * a.heads + lane.h) * a.cap + p;
      scale[i] = a.scale[which][row];
      *reinterpret_cast<uint2*>(c[i]) = *reinterpret_cast<const uint2*>(a.codes[which] + row * D + lane.at);
    }
    lane.next(a.heads);
  }
#pragma unroll
  for (int i = 0; i < KV_EACH; i++) {
    const unsigned v = lane.first + i * KvLane<D>::PER_WARP;
    if (v >= vectors) break;
    T* dst = static_cast<T*>(a.dst[which]) + ((int64_t)b * vectors + v) * D + lane.at;
#pragma unroll
    for (int e = 0; e < 2; e++) {
      uint32_t lo, hi;
      codes_to_half2<FMT>(c[i][e], lo, hi);
      float2 x = __half22float2(*reinterpret_cast<const __half2*>(&lo));
      float2 y = __half22float2(*reinterpret_cast<const __half2*>(&hi));
      x.x *= scale[i];
      x.y *= scale[i];
      y.x *= scale[i];
      y.y *= scale[i];
      if constexpr (sizeof(T) == 4) {
        reinterpret_cast<float4*>(dst)[e] = make_float4(x.x, x.y, y.x, y.y);
      } else if constexpr (std::is_same<T, __half>::value) {
        const __half2 v[2] = {__floats2half2_rn(x.x, x.y), __floats2half2_rn(y.x, y.y)};
        reinterpret_cast<uint2*>(dst)[e] = *reinterpret_cast<const uint2*>(v);
      } else {
        const __nv_bfloat162 v[2] = {__floats2bfloat162_rn(x.x, x.y), __floats2bfloat162_rn(y.x, y.y)};
        reinterpret_cast<uint2*>(dst)[e] = *reinterpret_cast<const uint2*>(v);
      }
    }
  }
}

// The attention layer's step between its projection and its attention (heads 256 wide): queries and keys normalised and
// rotated, queries rounded to fp16, keys and values quantised into the cache. One warp per vector: first the queries,
// then keys and values in turn. The vector passes through shared memory once, for the rotation's pairs.
struct QkvArgs {
  const float* qkv;
  int64_t stride;
  const float *qw, *kw;
  float eps, theta;
  int rot, nq, nkv, tokens;
  const int32_t* start;
  int64_t start_stride;
  __half* q;
  uint8_t* codes[2];
  float* scale[2];
  int64_t cap;
  int* err;
};

template <int FMT>
__global__ void __launch_bounds__(32 * KV_WARPS) qkv_append_kernel(const QkvArgs a) {
  constexpr int D = 256, N = D / 32;
  __shared__ __align__(16) float vec[KV_WARPS][D];
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int v = blockIdx.x * KV_WARPS + warp;  // 0 .. nq - 1: queries; then k0, v0, k1, v1, ..
  if (v >= a.nq + 2 * a.nkv) return;
  const int64_t row = blockIdx.y;  // sequence and token
  const int b = (int)(row / a.tokens), t = (int)(row % a.tokens);
  const bool query = v < a.nq;
  const int h = query ? v : (v - a.nq) / 2, which = query ? 0 : (v - a.nq) % 2;
  const float* src = a.qkv + row * a.stride +
                     (query ? (int64_t)h * 2 * D : (int64_t)a.nq * 2 * D + ((int64_t)which * a.nkv + h) * D) + lane * N;
  float f[N];
#pragma unroll
  for (int i = 0; i < N; i++) f[i] = src[i];
  const int64_t p = (int64_t)a.start[(int64_t)b * a.start_stride] + t;
  if (query || which == 0) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < N; i++) ss = fmaf(f[i], f[i], ss);
#pragma unroll
    for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float inv = rsqrtf(ss / D + a.eps);
    const float* w = (query ? a.qw : a.kw) + lane * N;
#pragma unroll
    for (int i = 0; i < N; i++) vec[warp][lane * N + i] = f[i] = f[i] * inv * w[i];
    __syncwarp();
    const int half = a.rot / 2;
#pragma unroll
    for (int i = 0; i < N; i++) {
      const int d = lane * N + i;
      if (d < a.rot) {
        const float ang = (float)p * powf(a.theta, -2.f * (float)(d % half) / (float)a.rot);
        float sn, cs;
        sincosf(ang, &sn, &cs);
        f[i] = f[i] * cs + (d < half ? -vec[warp][d + half] : vec[warp][d - half]) * sn;
      }
    }
  }
  if (query) {
    alignas(16) __half2 q[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; i++) q[i] = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
    *reinterpret_cast<uint4*>(a.q + (row * a.nq + h) * D + lane * N) = *reinterpret_cast<const uint4*>(q);
  } else if (p >= 0 && p < a.cap) {
    uint32_t code[N / 4];
    float scale;
    quantise<FMT, N>(f, code, scale);
    const int64_t at = ((int64_t)b * a.nkv + h) * a.cap + p;
    *reinterpret_cast<uint2*>(a.codes[which] + at * D + lane * N) = make_uint2(code[0], code[1]);
    if (lane == 0) a.scale[which][at] = scale;
  } else if (lane == 0 && a.err) {
    atomicExch(a.err, DEV_CACHE_POSITION);
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

// CTAs for `vectors` vectors of keys and of values in each sequence.
dim3 kv_grid(int64_t vectors, int64_t batch, int64_t dim) {
  const int64_t each = KV_WARPS * KV_EACH * (256 / dim);
  return dim3((unsigned)((vectors + each - 1) / each), (unsigned)batch, 2);
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
  if (tokens < 0 || tokens * heads > (1ll << 30)) return fail(GSQ_ERR_SIZE, "gsq_kv_append: bad token count");
  if (batch == 0 || tokens == 0) return GSQ_OK;
  if (!k || !v || !start || !k_strides || !v_strides) return fail(GSQ_ERR_ARG, "gsq_kv_append: null pointer");
  if (!words_aligned({start, counts})) return fail(GSQ_ERR_ALIGN, "gsq_kv_append: start or counts not aligned");
  const int64_t size = dtype == DT_F32 ? 4 : 2;
  KvArgs a = {};
  a.src[0] = k;
  a.src[1] = v;
  // vector loads where every vector starts on a 16-byte boundary
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
  a.tokens = (int)tokens;
  a.heads = (int)heads;
  a.cap = cap;
  a.err = device_error_word();
  const dim3 grid = kv_grid(tokens * heads, batch, dim);
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
  if (tokens < 0 || tokens * heads > (1ll << 30)) return fail(GSQ_ERR_SIZE, "gsq_kv_read: bad token count");
  if (batch == 0 || tokens == 0) return GSQ_OK;
  if (!k || !v || !start) return fail(GSQ_ERR_ARG, "gsq_kv_read: null pointer");
  if (!al16(k) || !al16(v) || !words_aligned({start, counts}))
    return fail(GSQ_ERR_ALIGN, "gsq_kv_read: outputs not 16-byte aligned, or start or counts not aligned");
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
  a.tokens = (int)tokens;
  a.heads = (int)heads;
  a.cap = cap;
  const dim3 grid = kv_grid(tokens * heads, batch, dim);
  cudaStream_t st = (cudaStream_t)stream;
  const cudaError_t e = fmt == KV_INT8 ? (dim == 256 ? read_launch<KV_INT8, 256>(dtype, grid, st, a)
                                                     : read_launch<KV_INT8, 128>(dtype, grid, st, a))
                                       : (dim == 256 ? read_launch<KV_FP8, 256>(dtype, grid, st, a)
                                                     : read_launch<KV_FP8, 128>(dtype, grid, st, a));
  return launched(e, "gsq_kv_read");
}

int gsq_qkv_append(const float* qkv, int64_t qkv_stride, int64_t batch, int64_t tokens, int64_t nq, int64_t nkv,
                   const float* q_norm_w, const float* k_norm_w, float eps, int64_t rot, float theta,
                   const int32_t* start, int64_t start_stride, void* q, int fmt, void* k_codes, void* v_codes,
                   float* k_scale, float* v_scale, int64_t cap, gsq_stream_t stream) {
  int rc = kv_check("gsq_qkv_append", fmt, k_codes, v_codes, k_scale, v_scale, batch, nkv, 256, cap);
  if (rc) return rc;
  if (tokens < 0 || batch * tokens > 65535) return fail(GSQ_ERR_SIZE, "gsq_qkv_append: at most 65535 tokens in all");
  if (nq <= 0 || nq > 65535 || qkv_stride < 512 * nq + 512 * nkv)
    return fail(GSQ_ERR_SIZE, "gsq_qkv_append: bad head count or stride");
  if (rot < 0 || rot > 256 || rot % 2) return fail(GSQ_ERR_SIZE, "gsq_qkv_append: bad rotary width");
  if (batch == 0 || tokens == 0) return GSQ_OK;
  if (!qkv || !q_norm_w || !k_norm_w || !start || !q) return fail(GSQ_ERR_ARG, "gsq_qkv_append: null pointer");
  if (!al16(q) || !words_aligned({qkv, q_norm_w, k_norm_w, start}))
    return fail(GSQ_ERR_ALIGN, "gsq_qkv_append: q not 16-byte aligned, or 4-byte values not aligned");
  QkvArgs a = {};
  a.qkv = qkv;
  a.stride = qkv_stride;
  a.qw = q_norm_w;
  a.kw = k_norm_w;
  a.eps = eps;
  a.theta = theta;
  a.rot = (int)rot;
  a.nq = (int)nq;
  a.nkv = (int)nkv;
  a.tokens = (int)tokens;
  a.start = start;
  a.start_stride = start_stride;
  a.q = static_cast<__half*>(q);
  a.codes[0] = static_cast<uint8_t*>(k_codes);
  a.codes[1] = static_cast<uint8_t*>(v_codes);
  a.scale[0] = k_scale;
  a.scale[1] = v_scale;
  a.cap = cap;
  a.err = device_error_word();
  const dim3 grid((unsigned)((nq + 2 * nkv + KV_WARPS - 1) / KV_WARPS), (unsigned)(batch * tokens));
  return launched(launch_pdl(fmt == KV_INT8 ? qkv_append_kernel<KV_INT8> : qkv_append_kernel<KV_FP8>, grid,
                             dim3(32 * KV_WARPS), 0, (cudaStream_t)stream, a),
                  "gsq_qkv_append");
}

}  // extern "C"
