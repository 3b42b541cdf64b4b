// mxq_kv.cu -- the paged 8-bit K/V cache: block tables and slot maps from
// request lengths, pages given back, new rows quantised into their blocks,
// cached tokens read back.
//
// The values are mx_quantize_x's (nn/core/layers/ssm.cpp:164-177: a shared
// power-of-two exponent and round-half-to-even int8), with the 32-element
// block laid over 32 tokens of one head instead of 32 features of a token.
#include "mxq_serve.cuh"

namespace mxq {

namespace {

// ------------------------------------------------------------------ plan --

struct PlanArgs {
  const int32_t *past, *add, *free_pages, *free_count;
  int32_t *table, *ctx_len, *cu, *slot, *position, *request, *free_out, *short_out;
  int R, P, max_pages, n_pages, N;
  uint32_t* done;
};

__device__ __forceinline__ int at_least_0(int x) { return x > 0 ? x : 0; }

// Largest i in [0, n) with a[i] <= x, for ascending a with a[0] <= x.
__device__ __forceinline__ int last_not_above(const int* a, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Inclusive sum over the block of one value a thread; every thread calls it.
__device__ __forceinline__ int block_scan(int v, int* warp_sums, int* total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  __syncthreads();                 // the sums of the last call have been read
  if (lane == 31) warp_sums[w] = v;
  __syncthreads();
  int before = 0, all = 0;
  for (int i = 0; i < nw; ++i) {
    if (i < w) before += warp_sums[i];
    all += warp_sums[i];
  }
  *total = all;
  return v + before;
}

// Every CTA sums the lengths itself (R ints from L2; a scan shared through
// memory would cost a second launch or a wait on another CTA) and then writes
// its share of the rows and of the new table entries.  What may be updated in
// place (the lengths, the stack's height) is written by the last CTA to
// finish, when the others have read it.
__global__ void __launch_bounds__(1024) kv_plan_kernel(PlanArgs a) {
  extern __shared__ int sh[];
  int* cu = sh;                    // [R + 1] first new row of a request
  int* pf = sh + a.R + 1;          // [R + 1] pages taken before it
  __shared__ int sums[32], sums2[32];
  __shared__ int missing;
  __shared__ int last;
  const int tid = threadIdx.x, nt = blockDim.x;
  if (tid == 0) missing = 0;
  int base_n = 0, base_p = 0, over = 0;
  for (int r0 = 0; r0 < a.R; r0 += nt) {
    const int r = r0 + tid;
    int n = 0, w = 0;
    if (r < a.R) {
      const int p = at_least_0(a.past[r]);
      n = at_least_0(a.add[r]);
      const int have = (p + a.P - 1) / a.P, full = (p + n + a.P - 1) / a.P;
      w = min(full, a.max_pages) - min(have, a.max_pages);
      over += full - have - w;     // pages beyond the table's width
    }
    int tn, tp;
    const int sn = block_scan(n, sums, &tn), sp = block_scan(w, sums2, &tp);
    if (r < a.R) {
      cu[r] = base_n + sn - n;
      pf[r] = base_p + sp - w;
    }
    base_n += tn;
    base_p += tp;
  }
  if (tid == 0) {
    cu[a.R] = base_n;
    pf[a.R] = base_p;
  }
  __syncthreads();
  if (over) atomicAdd(&missing, over);
  const int height = min(at_least_0(*a.free_count), a.n_pages);
  const int taken = min(base_p, height);
  const int t0 = blockIdx.x * nt + tid, step = gridDim.x * nt;

  for (int j = t0; j < base_p; j += step) {
    const int r = last_not_above(pf, a.R, j);
    const int have = (at_least_0(a.past[r]) + a.P - 1) / a.P;
    const int at = height - 1 - j;
    a.table[(long)r * a.max_pages + have + (j - pf[r])] = at >= 0 ? a.free_pages[at] : -1;
  }
  for (int i = t0; i < a.N; i += step) {
    int slot = -1, pos = -1, req = -1;
    if (i < base_n) {
      req = last_not_above(cu, a.R, i);
      const int p = at_least_0(a.past[req]);
      pos = p + (i - cu[req]);
      const int have = (p + a.P - 1) / a.P, pi = pos / a.P;
      if (pi < a.max_pages) {
        int page;
        if (pi < have) page = a.table[(long)req * a.max_pages + pi];
        else {
          const int at = height - 1 - (pf[req] + pi - have);
          page = at >= 0 ? a.free_pages[at] : -1;
        }
        if (page >= 0 && page < a.n_pages) slot = page * a.P + (pos - pi * a.P);
      }
    }
    a.slot[i] = slot;
    a.position[i] = pos;
    a.request[i] = req;
  }
  if (blockIdx.x == 0)
    for (int r = tid; r <= a.R; r += nt) a.cu[r] = cu[r];

  __syncthreads();
  if (tid == 0) {
    last = 1;
    if (gridDim.x > 1) {
      __threadfence();
      last = atomicAdd(a.done, 1u) == gridDim.x - 1;
      if (last) *a.done = 0;
    }
  }
  __syncthreads();
  if (!last) return;
  // lengths: past and its successor may be the same array, so each is read and written by one thread
  for (int r = tid; r < a.R; r += nt) a.ctx_len[r] = at_least_0(a.past[r]) + (cu[r + 1] - cu[r]);
  if (tid == 0) {
    *a.free_out = height - taken;
    *a.short_out = base_p - taken + missing;
  }
}

// --------------------------------------------------------------- release --

// One CTA: ending requests are few and their pages a few thousand; the order
// on the stack is fixed by a scan, not by which thread came first.
__global__ void __launch_bounds__(1024) kv_release_kernel(const uint8_t* done, int32_t* len, int R, int P,
                                                          int32_t* table, int max_pages, int32_t* free_pages,
                                                          int n_pages, int32_t* free_count) {
  extern __shared__ int pf[];      // [R + 1] pages of ended requests before this one
  __shared__ int sums[32];
  const int tid = threadIdx.x, nt = blockDim.x;
  int base = 0;
  for (int r0 = 0; r0 < R; r0 += nt) {
    const int r = r0 + tid;
    const int w = r < R && done[r] ? min((at_least_0(len[r]) + P - 1) / P, max_pages) : 0;
    int total;
    const int s = block_scan(w, sums, &total);
    if (r < R) pf[r] = base + s - w;
    base += total;
  }
  if (tid == 0) pf[R] = base;
  __syncthreads();
  int height = min(at_least_0(*free_count), n_pages);
  for (int j0 = 0; j0 < base; j0 += nt) {
    const int j = j0 + tid;
    int page = -1;
    if (j < base) {
      const int r = last_not_above(pf, R, j);
      int32_t* e = table + (long)r * max_pages + (j - pf[r]);
      page = *e;
      *e = -1;
      if (page >= n_pages) page = -1;
    }
    int total;
    const int s = block_scan(page >= 0, sums, &total);
    if (page >= 0 && height + s - 1 < n_pages) free_pages[height + s - 1] = page;
    height = min(height + total, n_pages);
  }
  __syncthreads();
  if (tid == 0) *free_count = height;
  for (int r = tid; r < R; r += nt)
    if (done[r]) len[r] = 0;
}

// ---------------------------------------------------------------- append --

constexpr int kAppendThreads = 256;
constexpr int kCtaRun = 8;         // runs of at least this many rows take the whole CTA, shorter ones a warp

// Four int8 of a word re-rounded to a step 2^d times as large.
__device__ __forceinline__ uint32_t reround4(uint32_t w, float down) {
  uint32_t r = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int q = __float2int_rn((float)(int8_t)(w >> (8 * i)) * down);
    r |= (uint32_t)(q & 0xFF) << (8 * i);
  }
  return r;
}
__device__ __forceinline__ uint4 reround16(uint4 w, float down) {
  return make_uint4(reround4(w.x, down), reround4(w.y, down), reround4(w.z, down), reround4(w.w, down));
}

// Scale byte of the largest |x| given as bits (NaN and inf are above every finite one).
__device__ __forceinline__ int scale_byte(uint32_t top) {
  return top >= 0x7f800000u ? 255 : e8m0_exponent<127>(__uint_as_float(top)) + 127;
}
__device__ __forceinline__ int quant_byte(float x, int byte) {
  return byte == 255 ? 0 : quant_value(x, byte - 127);
}
// 2^(from - to), 0 once every int8 rounds to 0
__device__ __forceinline__ float step_down(int from, int to) {
  const int d = to - from;
  return d > 30 ? 0.0f : __int_as_float((127 - d) << 23);
}

// One CTA: the runs that start in `chunk` consecutive rows, of one head, of K
// (z = 0) or V (z = 1).  A run of a prompt fills up to 32 rows: 256 threads
// hold it in registers, agree on the exponent, and write 16 bytes each (V by
// way of shared memory, which turns it).  A decode step's runs are one row
// each: a warp a run.
template <typename T, int D>
__global__ void __launch_bounds__(kAppendThreads)
    kv_append_kernel(KvView c, const T* __restrict__ k, const T* __restrict__ v, long stride,
                     const int32_t* __restrict__ slot, int n, int chunk) {
  constexpr int kPad = 4;
  __shared__ int s_slot[32 + 33];
  __shared__ int s_first[32], s_len[32];
  __shared__ int s_runs;
  __shared__ uint32_t s_top[kAppendThreads / 32];
  __shared__ uint8_t s_q[32][D + kPad];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int base = blockIdx.x * chunk, head = blockIdx.y;
  const bool is_v = blockIdx.z != 0;
  const T* src = (is_v ? v : k) + (long)head * D;
  int8_t* data = is_v ? c.v : c.k;
  uint8_t* scales = is_v ? c.vs : c.ks;
  const int slots = c.n_pages * c.page;

  // slots of the rows base - 1 .. base + chunk + 30
  for (int i = tid; i < chunk + 32; i += kAppendThreads) {
    const int row = base - 1 + i;
    const int s = row >= 0 && row < n ? slot[row] : -1;
    s_slot[i] = s >= 0 && s < slots ? s : -1;
  }
  __syncthreads();
  if (warp == 0) {
    bool lead = false;
    int len = 0;
    if (lane < chunk) {
      const int s = s_slot[lane + 1], before = s_slot[lane];
      lead = s >= 0 && (before < 0 || (before >> 5) != (s >> 5));
      if (lead)
        for (len = 1; len < 32; ++len) {
          const int u = s_slot[lane + 1 + len];
          if (u < 0 || (u >> 5) != (s >> 5)) break;
        }
    }
    const uint32_t all = __ballot_sync(0xffffffffu, lead);
    if (lead) {
      const int at = __popc(all & ((1u << lane) - 1));
      s_first[at] = lane;
      s_len[at] = len;
    }
    if (lane == 0) s_runs = __popc(all);
  }
  __syncthreads();
  const int runs = s_runs;

  for (int i = 0; i < runs; ++i) {           // long runs: the whole CTA
    const int first = s_first[i], len = s_len[i];
    if (len < kCtaRun) continue;
    const int s0 = s_slot[first + 1];
    const long blk = kv_block(c, s0 / c.page, head, (s0 % c.page) >> 5);
    uint8_t* dst = reinterpret_cast<uint8_t*>(data) + blk * (32 * D);
    constexpr int kVals = D / 8;             // values a thread: row tid / 8, an eighth of it
    const int row = tid >> 3, seg = tid & 7;
    float x[kVals];
    uint32_t top = 0;
    if (row < len) {
#pragma unroll
      for (int u = 0; u < kVals; u += 4) {
        float y[4];
        load4(src + (long)(base + first + row) * stride + seg * kVals + u, y);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[u + e] = y[e];
          top = max(top, __float_as_uint(y[e]) & 0x7fffffffu);
        }
      }
    }
    const bool extends = (s0 & 31) != 0;
    const int was = extends ? scales[blk] : 0;
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) s_top[warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kAppendThreads / 32; ++w) top = max(top, s_top[w]);
    const int byte = max(scale_byte(top), was);
    const bool grew = extends && byte > was && byte != 255;
    const float down = grew ? step_down(was, byte) : 1.0f;
    uint32_t in_run = 0;
    for (int r = 0; r < len; ++r) in_run |= 1u << (s_slot[first + 1 + r] & 31);
    uint32_t q[kVals / 4];
    if (row < len) {
#pragma unroll
      for (int u = 0; u < kVals; ++u) {
        if ((u & 3) == 0) q[u / 4] = 0;
        q[u / 4] |= (uint32_t)(quant_byte(x[u], byte) & 0xFF) << (8 * (u & 3));
      }
      const int t = s_slot[first + 1 + row] & 31;
      uint8_t* to = is_v ? &s_q[t][seg * kVals] : dst + t * D + seg * kVals;
#pragma unroll
      for (int u = 0; u < kVals / 4; ++u) reinterpret_cast<uint32_t*>(to)[u] = q[u];
    }
    if (!is_v) {
      if (grew && !(in_run >> row & 1)) {
        uint32_t* old = reinterpret_cast<uint32_t*>(dst + row * D + seg * kVals);
#pragma unroll
        for (int u = 0; u < kVals / 4; ++u) old[u] = reround4(old[u], down);
      }
    } else {
      __syncthreads();
      for (int ch = tid; ch < 2 * D; ch += kAppendThreads) {   // 16 bytes: two dimensions, eight tokens
        const int pair = ch >> 2, cc = ch & 3;
        uint4* to = reinterpret_cast<uint4*>(dst) + ch;
        uint4 w = make_uint4(0, 0, 0, 0);
        if (extends) {
          w = *to;
          if (grew) w = reround16(w, down);
        }
        uint32_t out[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int dd = e >> 3, t = ((e & 7) >> 1) * 8 + 2 * cc + (e & 1);
          if (in_run >> t & 1) {
            const uint32_t b = s_q[t][2 * pair + dd];
            out[e >> 2] = (out[e >> 2] & ~(0xFFu << (8 * (e & 3)))) | b << (8 * (e & 3));
          }
        }
        *to = make_uint4(out[0], out[1], out[2], out[3]);
      }
    }
    if (tid == 0) scales[blk] = (uint8_t)byte;
    __syncthreads();
  }

  for (int i = warp; i < runs; i += kAppendThreads / 32) {   // short runs: a warp each
    const int first = s_first[i], len = s_len[i];
    if (len >= kCtaRun) continue;
    const int s0 = s_slot[first + 1];
    const long blk = kv_block(c, s0 / c.page, head, (s0 % c.page) >> 5);
    uint8_t* dst = reinterpret_cast<uint8_t*>(data) + blk * (32 * D);
    const bool extends = (s0 & 31) != 0, mine = lane < D / 4;
    const int was = extends ? scales[blk] : 0;
    uint32_t top = 0;
    if (mine)
      for (int r = 0; r < len; ++r) {
        float y[4];
        load4(src + (long)(base + first + r) * stride + lane * 4, y);
#pragma unroll
        for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(y[e]) & 0x7fffffffu);
      }
    top = __reduce_max_sync(0xffffffffu, top);
    const int byte = max(scale_byte(top), was);
    if (extends && byte > was && byte != 255) {
      const float down = step_down(was, byte);
#pragma unroll
      for (int u = 0; u < 2 * D / 32; ++u) {
        uint4* w = reinterpret_cast<uint4*>(dst) + u * 32 + lane;
        *w = reround16(*w, down);
      }
      __syncwarp();
    }
    if (mine)
      for (int r = 0; r < len; ++r) {
        float y[4];
        load4(src + (long)(base + first + r) * stride + lane * 4, y);
        const int t = s_slot[first + 1 + r] & 31;
        uint32_t w = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t q = (uint32_t)quant_byte(y[e], byte) & 0xFF;
          if (is_v) dst[v_offset(t, lane * 4 + e)] = (uint8_t)q;
          w |= q << (8 * e);
        }
        if (!is_v) *reinterpret_cast<uint32_t*>(dst + t * D + lane * 4) = w;
      }
    if (lane == 0) scales[blk] = (uint8_t)byte;
  }
}

// ------------------------------------------------------------------ read --

template <typename T, int D>
__global__ void __launch_bounds__(256) kv_read_kernel(KvView c, const int32_t* __restrict__ slot, int n,
                                                      T* __restrict__ k_out, T* __restrict__ v_out) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, head = blockIdx.y;
  const bool is_v = blockIdx.z != 0;
  if (lane >= D / 4) return;
  for (int i = blockIdx.x * 32 + warp; i < min(n, (int)(blockIdx.x + 1) * 32); i += 8) {
    const int s = slot[i];
    float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (s >= 0 && s < c.n_pages * c.page) {
      const long blk = kv_block(c, s / c.page, head, (s % c.page) >> 5);
      const int8_t* at = (is_v ? c.v : c.k) + blk * (32 * D);
      const float sc = e8m0_to_float((is_v ? c.vs : c.ks)[blk]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = lane * 4 + e;
        y[e] = (float)at[is_v ? v_offset(s & 31, d) : (s & 31) * D + d] * sc;
      }
    }
    store4((is_v ? v_out : k_out) + ((long)i * c.heads + head) * D + lane * 4, y);
  }
}

template <typename T>
cudaError_t launch_append(const KvView& c, const void* k, const void* v, long stride, const int32_t* slot, int n,
                          cudaStream_t st) {
  // 8 rows a CTA while that leaves the GPU with few of them, 32 beyond
  const int chunk = (long)n * c.heads <= 8l * 148 * 8 ? 8 : 32;
  const dim3 grid((unsigned)((n + chunk - 1) / chunk), (unsigned)c.heads, 2);
  if (c.dim == 64)
    kv_append_kernel<T, 64><<<grid, kAppendThreads, 0, st>>>(c, static_cast<const T*>(k), static_cast<const T*>(v),
                                                             stride, slot, n, chunk);
  else
    kv_append_kernel<T, 128><<<grid, kAppendThreads, 0, st>>>(c, static_cast<const T*>(k), static_cast<const T*>(v),
                                                              stride, slot, n, chunk);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_read(const KvView& c, const int32_t* slot, int n, void* k, void* v, cudaStream_t st) {
  const dim3 grid((unsigned)((n + 31) / 32), (unsigned)c.heads, 2);
  if (c.dim == 64)
    kv_read_kernel<T, 64><<<grid, 256, 0, st>>>(c, slot, n, static_cast<T*>(k), static_cast<T*>(v));
  else
    kv_read_kernel<T, 128><<<grid, 256, 0, st>>>(c, slot, n, static_cast<T*>(k), static_cast<T*>(v));
  return cudaGetLastError();
}

SmemAttr g_plan_attr, g_release_attr;

int bad(mxq_context* c, const char* msg) { return ctx_fail(c, MXQ_ERR_INVALID_ARGUMENT, msg); }

}  // namespace
}  // namespace mxq

using namespace mxq;

extern "C" {

int mxq_kv_plan(mxq_ctx c, const int32_t* past, const int32_t* add, size_t n_req, size_t page_size, int32_t* table,
                size_t max_pages, const int32_t* free_pages, size_t n_pages, const int32_t* free_count,
                int32_t* ctx_len, int32_t* cu, int32_t* slot, int32_t* position, int32_t* request, size_t n_tokens,
                int32_t* free_out, int32_t* short_out) {
  if (!c) return bad(nullptr, "null context");
  if (!past || !add || !table || !free_pages || !free_count || !ctx_len || !cu || !free_out || !short_out ||
      (n_tokens && (!slot || !position || !request)))
    return bad(c, "kv plan: null pointer");
  if (n_req == 0 || n_req > MXQ_KV_MAX_REQUESTS) return bad(c, "kv plan: 1 to 8192 requests");
  if (page_size < kBlock || page_size > 1024 || page_size % kBlock)
    return bad(c, "kv plan: the page size is a multiple of 32, at most 1024");
  if (max_pages == 0 || max_pages > (1u << 26) || n_pages == 0 || n_pages * page_size >= (1ull << 31))
    return bad(c, "kv plan: bad number of pages");
  if (n_tokens > (1u << 30)) return bad(c, "kv plan: too many new tokens");
  ServeDevice g(ctx_device(c));
  ServeWs ws;
  if (int rc = ctx_serve_ws(c, &ws)) return rc;
  PlanArgs a{past, add, free_pages, free_count, table, ctx_len, cu, slot, position, request, free_out, short_out,
             (int)n_req, (int)page_size, (int)max_pages, (int)n_pages, (int)n_tokens, ws.counters};
  // a thread a new row up to 4 CTAs an SM; small steps in one CTA of 256
  const size_t most = n_tokens > n_req ? n_tokens : n_req;
  const int threads = most <= 4096 ? 256 : 1024;
  size_t ctas = (most + threads - 1) / threads;
  if (ctas > (size_t)ws.sms) ctas = (size_t)ws.sms;
  const size_t smem = 2 * (n_req + 1) * sizeof(int);
  cudaError_t e = g_plan_attr.ensure(kv_plan_kernel, smem);
  if (e == cudaSuccess) {
    kv_plan_kernel<<<(unsigned)ctas, threads, smem, ctx_stream(c)>>>(a);
    e = cudaGetLastError();
  }
  return serve_launched(c, e, "kv plan");
}

int mxq_kv_release(mxq_ctx c, const uint8_t* done, int32_t* len, size_t n_req, size_t page_size, int32_t* table,
                   size_t max_pages, int32_t* free_pages, size_t n_pages, int32_t* free_count) {
  if (!c) return bad(nullptr, "null context");
  if (!done || !len || !table || !free_pages || !free_count) return bad(c, "kv release: null pointer");
  if (n_req == 0 || n_req > MXQ_KV_MAX_REQUESTS) return bad(c, "kv release: 1 to 8192 requests");
  if (page_size < kBlock || page_size > 1024 || page_size % kBlock)
    return bad(c, "kv release: the page size is a multiple of 32, at most 1024");
  if (max_pages == 0 || max_pages > (1u << 26) || n_pages == 0 || n_pages * page_size >= (1ull << 31))
    return bad(c, "kv release: bad number of pages");
  ServeDevice g(ctx_device(c));
  const size_t smem = (n_req + 1) * sizeof(int);
  cudaError_t e = g_release_attr.ensure(kv_release_kernel, smem);
  if (e == cudaSuccess) {
    kv_release_kernel<<<1, 1024, smem, ctx_stream(c)>>>(done, len, (int)n_req, (int)page_size, table, (int)max_pages,
                                                        free_pages, (int)n_pages, free_count);
    e = cudaGetLastError();
  }
  return serve_launched(c, e, "kv release");
}

int mxq_kv_append(mxq_ctx c, const mxq_kv_cache* cache, int dtype, const void* k, const void* v, size_t row_stride,
                  const int32_t* slot, size_t n) {
  if (!c) return bad(nullptr, "null context");
  KvView kv;
  if (const char* msg = kv_view(cache, &kv)) return bad(c, msg);
  const size_t es = dtype_bytes(dtype);
  if (!es) return bad(c, "kv append: unknown row type");
  if (n == 0) return MXQ_OK;
  if (!k || !v || !slot) return bad(c, "kv append: null pointer");
  if (n > (1u << 30)) return bad(c, "kv append: too many rows");
  if (row_stride < (size_t)kv.heads * kv.dim) return bad(c, "kv append: rows overlap");
  if (!aligned16(k) || !aligned16(v) || row_stride * es % 16)
    return bad(c, "kv append: rows must start on 16-byte boundaries");
  ServeDevice g(ctx_device(c));
  const cudaStream_t st = ctx_stream(c);
  const cudaError_t e =
      dtype == MXQ_DT_F32 ? launch_append<float>(kv, k, v, (long)row_stride, slot, (int)n, st)
      : dtype == MXQ_DT_BF16 ? launch_append<__nv_bfloat16>(kv, k, v, (long)row_stride, slot, (int)n, st)
                             : launch_append<__half>(kv, k, v, (long)row_stride, slot, (int)n, st);
  return serve_launched(c, e, "kv append");
}

int mxq_kv_read(mxq_ctx c, const mxq_kv_cache* cache, const int32_t* slot, size_t n, int dtype, void* k_out,
                void* v_out) {
  if (!c) return bad(nullptr, "null context");
  KvView kv;
  if (const char* msg = kv_view(cache, &kv)) return bad(c, msg);
  if (!dtype_bytes(dtype)) return bad(c, "kv read: unknown row type");
  if (n == 0) return MXQ_OK;
  if (!slot || !k_out || !v_out) return bad(c, "kv read: null pointer");
  if (n > (1u << 30)) return bad(c, "kv read: too many rows");
  if (!aligned16(k_out) || !aligned16(v_out)) return bad(c, "kv read: outputs must be 16-byte aligned");
  ServeDevice g(ctx_device(c));
  const cudaStream_t st = ctx_stream(c);
  const cudaError_t e = dtype == MXQ_DT_F32    ? launch_read<float>(kv, slot, (int)n, k_out, v_out, st)
                        : dtype == MXQ_DT_BF16 ? launch_read<__nv_bfloat16>(kv, slot, (int)n, k_out, v_out, st)
                                               : launch_read<__half>(kv, slot, (int)n, k_out, v_out, st);
  return serve_launched(c, e, "kv read");
}

}  // extern "C"
