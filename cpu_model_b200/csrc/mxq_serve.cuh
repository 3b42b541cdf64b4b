// mxq_serve.cuh -- helpers shared by the serving kernels (mxq_kv.cu,
// mxq_kvattn.cu, mxq_logprob.cu): row types, the K/V cache's addressing and
// the host checks common to their entry points.
#pragma once
#include <cuda_fp16.h>

#include "mxq_internal.h"

namespace mxq {

// Where a K/V cache's blocks are (host view of mxq_kv_cache).
struct KvView {
  int8_t* k;
  int8_t* v;
  uint8_t* ks;
  uint8_t* vs;
  int n_pages, page, nb, heads, dim;   // nb: blocks a page
};

// Attention of the requests with more than `few` query rows a K/V head, 16-bit
// rows (mxq_kvprompt.cu).
struct KvPromptArgs {
  KvView c;
  const void* q;
  void* out;
  float* lse;
  const int32_t *table, *ctx_len, *cu;
  long q_stride;
  int R, n, Hq, G, max_pages, few, bf16;
  float scale2;                          // scale * log2(e)
  uint32_t* next;                        // two words, zero
  uint32_t* status;
};
cudaError_t launch_kv_prompt(const KvPromptArgs& a, int ctas, cudaStream_t st);

constexpr float kLn2 = 0.693147180559945f, kLog2e = 1.44269504088896341f;
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float neg_inf() { return -__int_as_float(0x7f800000); }

// Index of (page, head, block of the page): its scale's place; its values
// start at 32 * dim times it.
__device__ __forceinline__ long kv_block(const KvView& c, int page, int head, int b) {
  return ((long)page * c.heads + head) * c.nb + b;
}

// Byte of (token t, dimension d) inside a V block.
__host__ __device__ __forceinline__ int v_offset(int t, int d) {
  return ((d >> 1) * 4 + ((t >> 1) & 3)) * 16 + (d & 1) * 8 + (t >> 3) * 2 + (t & 1);
}

// ceil(x / d), 0 for x < 0: for every int x (x + d - 1 may not be one).
__host__ __device__ __forceinline__ int ceil_div(int x, int d) {
  return x > 0 ? (int)(((unsigned)x + (unsigned)d - 1) / (unsigned)d) : 0;
}

// Keys and blocks of a request that its block table has places for: no more is
// looked at, however long the request says it is.
__device__ __forceinline__ int table_keys(const KvView& c, int max_pages, int len) {
  return (int)min((long)max_pages * c.page, (long)max(len, 0));
}

// ------------------------------------------------------------- row types --
template <typename T> __device__ __forceinline__ float to_f32(T x);
template <> __device__ __forceinline__ float to_f32(float x) { return x; }
template <> __device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }

template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_f32(float x) { return __float2half_rn(x); }

// Four consecutive elements (aligned to their size).
template <typename T> __device__ __forceinline__ void load4(const T* p, float (&v)[4]);
template <> __device__ __forceinline__ void load4(const float* p, float (&v)[4]) {
  const float4 x = *reinterpret_cast<const float4*>(p);
  v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
}
template <> __device__ __forceinline__ void load4(const __nv_bfloat16* p, float (&v)[4]) {
  const uint2 x = *reinterpret_cast<const uint2*>(p);
  v[0] = __uint_as_float(x.x << 16); v[1] = __uint_as_float(x.x & 0xFFFF0000u);
  v[2] = __uint_as_float(x.y << 16); v[3] = __uint_as_float(x.y & 0xFFFF0000u);
}
template <> __device__ __forceinline__ void load4(const __half* p, float (&v)[4]) {
  const uint2 x = *reinterpret_cast<const uint2*>(p);
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&x.x));
  const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&x.y));
  v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
}

template <typename T> __device__ __forceinline__ void store4(T* p, const float (&v)[4]);
template <> __device__ __forceinline__ void store4(float* p, const float (&v)[4]) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
template <> __device__ __forceinline__ void store4(__nv_bfloat16* p, const float (&v)[4]) {
  const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
  *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}
template <> __device__ __forceinline__ void store4(__half* p, const float (&v)[4]) {
  const __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
  *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

// Row types whose kind is known at run time only (a few rows a call).
__device__ __forceinline__ void load4_dt(int dt, const void* p, long at, float (&v)[4]) {
  if (dt == MXQ_DT_F32) load4(static_cast<const float*>(p) + at, v);
  else if (dt == MXQ_DT_BF16) load4(static_cast<const __nv_bfloat16*>(p) + at, v);
  else load4(static_cast<const __half*>(p) + at, v);
}
__device__ __forceinline__ void store4_dt(int dt, void* p, long at, const float (&v)[4]) {
  if (dt == MXQ_DT_F32) store4(static_cast<float*>(p) + at, v);
  else if (dt == MXQ_DT_BF16) store4(static_cast<__nv_bfloat16*>(p) + at, v);
  else store4(static_cast<__half*>(p) + at, v);
}

__device__ __forceinline__ void store2_dt(int dt, void* p, long at, float x, float y) {
  if (dt == MXQ_DT_F32) *reinterpret_cast<float2*>(static_cast<float*>(p) + at) = make_float2(x, y);
  else if (dt == MXQ_DT_BF16)
    *reinterpret_cast<__nv_bfloat162*>(static_cast<__nv_bfloat16*>(p) + at) = __floats2bfloat162_rn(x, y);
  else *reinterpret_cast<__half2*>(static_cast<__half*>(p) + at) = __floats2half2_rn(x, y);
}

// ------------------------------------------------------------------ host --
struct ServeDevice {
  int prev = -1;
  explicit ServeDevice(int dev) {
    if (cudaGetDevice(&prev) == cudaSuccess && prev != dev) cudaSetDevice(dev);
    else prev = -1;
  }
  ~ServeDevice() {
    if (prev >= 0) cudaSetDevice(prev);
  }
};

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Checks a cache descriptor; null when it is sound, else what is wrong.
inline const char* kv_view(const mxq_kv_cache* c, KvView* v) {
  if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale) return "kv cache: null pointer";
  if (c->n_pages <= 0 || c->n_kv_heads <= 0 || c->n_kv_heads > 1024) return "kv cache: bad number of pages or heads";
  if (c->page_size < kBlock || c->page_size > 1024 || c->page_size % kBlock)
    return "kv cache: the page size is a multiple of 32, at most 1024";
  if (c->head_dim != 64 && c->head_dim != 128) return "kv cache: the head dimension is 64 or 128";
  if ((long)c->n_pages * c->page_size >= (1l << 31)) return "kv cache: more than 2^31 token slots";
  if (!aligned16(c->k) || !aligned16(c->v)) return "kv cache: k and v must be 16-byte aligned";
  *v = KvView{static_cast<int8_t*>(c->k), static_cast<int8_t*>(c->v), c->k_scale, c->v_scale,
              c->n_pages, c->page_size, c->page_size / kBlock, c->n_kv_heads, c->head_dim};
  return nullptr;
}

inline int serve_launched(mxq_context* c, cudaError_t e, const char* what) {
  if (e != cudaSuccess) return ctx_cuda_fail(c, e, what);
  ctx_add_launches(c, 1);
  return MXQ_OK;
}

}  // namespace mxq
