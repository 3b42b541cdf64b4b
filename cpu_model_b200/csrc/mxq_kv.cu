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

// Inclusive sums over the block of a pair of values a thread; every thread calls it.
__device__ __forceinline__ int2 block_scan(int2 v, int2* warp_sums, int2* total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, v.x, o), b = __shfl_up_sync(0xffffffffu, v.y, o);
    if (lane >= o) v.x += a, v.y += b;
  }
  __syncthreads();                 // the sums of the last call have been read
  if (lane == 31) warp_sums[w] = v;
  __syncthreads();
  int2 s = lane < nw ? warp_sums[lane] : make_int2(0, 0);
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, s.x, o), b = __shfl_up_sync(0xffffffffu, s.y, o);
    if (lane >= o) s.x += a, s.y += b;
  }
  const int before = w > 0 ? w - 1 : 0;
  const int bx = __shfl_sync(0xffffffffu, s.x, before), by = __shfl_sync(0xffffffffu, s.y, before);
  if (w > 0) v.x += bx, v.y += by;
  *total = make_int2(__shfl_sync(0xffffffffu, s.x, 31), __shfl_sync(0xffffffffu, s.y, 31));
  return v;
}

// Every CTA sums the lengths itself (R ints from L2; a scan shared through
// memory would cost a second launch or a wait on another CTA), one scan over the
// threads with a few requests each, and then writes its share of the rows and
// of the new table entries.  What may be updated in place (the lengths, the
// stack's height) is written by the last CTA to finish, when the others have
// read it.  Bound by latency: 3.6 us for 32 requests of one token each, 10.4 us for
// 4096 requests with 88.7k rows, of which the sums are most.
__global__ void __launch_bounds__(1024) kv_plan_kernel(PlanArgs a) {
  extern __shared__ int sh[];
  int* cu = sh;                    // [R + 1] first new row of a request
  int* pf = cu + a.R + 1;          // [R + 1] pages taken before it
  int* len = pf + a.R + 1;         // [R] its past
  __shared__ int2 sums[32];
  __shared__ int missing;
  __shared__ int last;
  const int tid = threadIdx.x, nt = blockDim.x;
  const int height = min(at_least_0(*a.free_count), a.n_pages);
  if (tid == 0) missing = 0;
  for (int r = tid; r < a.R; r += nt) {
    len[r] = at_least_0(a.past[r]);
    cu[r] = at_least_0(a.add[r]);
  }
  __syncthreads();
  const int own = (a.R + nt - 1) / nt, r0 = min(tid * own, a.R), r1 = min(r0 + own, a.R);
  int over = 0;
  int2 mine = make_int2(0, 0);
  for (int r = r0; r < r1; ++r) {
    const int have = ceil_div(len[r], a.P), full = ceil_div(len[r] + cu[r], a.P);
    const int w = min(full, a.max_pages) - min(have, a.max_pages);
    over += full - have - w;       // pages beyond the table's width
    pf[r] = w;
    mine.x += cu[r];
    mine.y += w;
  }
  int2 all;
  const int2 upto = block_scan(mine, sums, &all);
  int2 at = make_int2(upto.x - mine.x, upto.y - mine.y);
  for (int r = r0; r < r1; ++r) {
    const int n = cu[r], w = pf[r];
    cu[r] = at.x;
    pf[r] = at.y;
    at.x += n;
    at.y += w;
  }
  if (tid == 0) {
    cu[a.R] = all.x;
    pf[a.R] = all.y;
  }
  if (over) atomicAdd(&missing, over);
  __syncthreads();
  const int rows = all.x, wanted = all.y, taken = min(wanted, height);
  const int t0 = blockIdx.x * nt + tid, step = gridDim.x * nt;

  for (int j = t0; j < wanted; j += step) {
    const int r = last_not_above(pf, a.R, j);
    const int have = ceil_div(len[r], a.P), from = height - 1 - j;
    a.table[(long)r * a.max_pages + have + (j - pf[r])] = from >= 0 ? a.free_pages[from] : -1;
  }
  for (int i = t0; i < a.N; i += step) {
    int slot = -1, pos = -1, req = -1;
    if (i < rows) {
      req = last_not_above(cu, a.R, i);
      const int p = len[req];
      pos = p + (i - cu[req]);
      const int have = ceil_div(p, a.P), pi = pos / a.P;
      if (pos >= 0 && pi < a.max_pages) {
        const int from = height - 1 - (pf[req] + pi - have);
        const int page = pi < have ? a.table[(long)req * a.max_pages + pi] : from >= 0 ? a.free_pages[from] : -1;
        if (page >= 0 && page < a.n_pages) slot = page * a.P + (pos - pi * a.P);
      }
    }
    a.slot[i] = slot;
    a.position[i] = pos;
    a.request[i] = req;
  }
  for (int r = t0; r <= a.R; r += step) a.cu[r] = cu[r];

  if (gridDim.x > 1) {
    __threadfence();
    __syncthreads();
    if (tid == 0) {
      last = atomicAdd(a.done, 1u) == gridDim.x - 1;
      if (last) *a.done = 0;
    }
    __syncthreads();
    if (!last) return;
  }
  for (int r = tid; r < a.R; r += nt) a.ctx_len[r] = len[r] + (cu[r + 1] - cu[r]);
  if (tid == 0) {
    *a.free_out = height - taken;
    *a.short_out = wanted - taken + missing;
  }
}

// --------------------------------------------------------------- release --

// One CTA, bound by latency: ending requests are few and their pages a few
// thousand; the order on the stack is fixed by a scan, not by which thread came first.
// 64 of 4096 requests with 20 pages each: 9 us.
__global__ void __launch_bounds__(1024) kv_release_kernel(const uint8_t* done, int32_t* len, int R, int P,
                                                          int32_t* table, int max_pages, int32_t* free_pages,
                                                          int n_pages, int32_t* free_count) {
  extern __shared__ int pf[];      // [R + 1] pages of ended requests before this one
  __shared__ int2 sums[32];
  const int tid = threadIdx.x, nt = blockDim.x;
  int base = 0;
  for (int r0 = 0; r0 < R; r0 += nt) {
    const int r = r0 + tid;
    const int w = r < R && done[r] ? min(ceil_div(len[r], P), max_pages) : 0;
    int2 total;
    const int s = block_scan(make_int2(w, 0), sums, &total).x;
    if (r < R) pf[r] = base + s - w;
    base += total.x;
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
    int2 total;
    const int s = block_scan(make_int2(page >= 0, 0), sums, &total).x;
    if (page >= 0 && height + s - 1 < n_pages) free_pages[height + s - 1] = page;
    height = min(height + total.x, n_pages);
  }
  __syncthreads();
  if (tid == 0) *free_count = height;
  for (int r = tid; r < R; r += nt)
    if (done[r]) len[r] = 0;
}

// ---------------------------------------------------------------- append --

constexpr int kCopyWarps = 4;      // warps a CTA, each on its own
constexpr int kLongRun = 8;        // runs of at least this many rows are built in registers

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
// 2^(from - to), 0 once every int8 rounds to 0
__device__ __forceinline__ float step_down(int from, int to) {
  const int d = to - from;
  return d > 30 ? 0.0f : __int_as_float((127 - d) << 23);
}
// rint(x * inv) in the low byte: x * inv is exact (a power of two), the sum with 1.5 * 2^23 rounds it half to even
__device__ __forceinline__ uint32_t quant_bits(float x, float inv) {
  return __float_as_uint(fmaf(x, inv, 12582912.0f));
}

// A lane's V consecutive values of a row, as loaded.
template <typename T, int V> struct Raw {
  uint32_t w[V * sizeof(T) / 4];
  __device__ __forceinline__ void load(const T* p) {
    constexpr int kBytes = V * (int)sizeof(T);
    if (kBytes == 16) {
      const uint4 x = __ldg(reinterpret_cast<const uint4*>(p));
      w[0] = x.x; w[1 % (kBytes / 4)] = x.y; w[2 % (kBytes / 4)] = x.z; w[3 % (kBytes / 4)] = x.w;
    } else if (kBytes == 8) {
      const uint2 x = __ldg(reinterpret_cast<const uint2*>(p));
      w[0] = x.x; w[1 % (kBytes / 4)] = x.y;
    } else {
      w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < V * (int)sizeof(T) / 4; ++i) w[i] = 0;
  }
  __device__ __forceinline__ float get(int i) const;
  // The largest |value| so far, in whatever order-keeping bits the type has; f32_bits() of it at the end.
  __device__ __forceinline__ uint32_t top(uint32_t so_far) const {
#pragma unroll
    for (int i = 0; i < V * (int)sizeof(T) / 4; ++i)
      so_far = sizeof(T) == 4 ? max(so_far, w[i] & 0x7fffffffu) : __vmaxu2(so_far, w[i] & 0x7fff7fffu);
    return so_far;
  }
};
// What Raw::top left, as the bits of an fp32 number.
template <typename T> __device__ __forceinline__ uint32_t f32_bits(uint32_t top);
template <> __device__ __forceinline__ uint32_t f32_bits<float>(uint32_t top) { return top; }
template <> __device__ __forceinline__ uint32_t f32_bits<__nv_bfloat16>(uint32_t top) { return max(top & 0xffffu, top >> 16) << 16; }
template <> __device__ __forceinline__ uint32_t f32_bits<__half>(uint32_t top) {
  return __float_as_uint(__half2float(__ushort_as_half((unsigned short)max(top & 0xffffu, top >> 16))));
}
template <> __device__ __forceinline__ float Raw<float, 4>::get(int i) const { return __uint_as_float(w[i]); }
template <> __device__ __forceinline__ float Raw<float, 2>::get(int i) const { return __uint_as_float(w[i]); }
__device__ __forceinline__ float bf16_at(uint32_t w, int i) { return __uint_as_float(i & 1 ? w & 0xFFFF0000u : w << 16); }
template <> __device__ __forceinline__ float Raw<__nv_bfloat16, 4>::get(int i) const { return bf16_at(w[i >> 1], i); }
template <> __device__ __forceinline__ float Raw<__nv_bfloat16, 2>::get(int i) const { return bf16_at(w[0], i); }
__device__ __forceinline__ float f16_at(uint32_t w, int i) {
  return __half2float(__ushort_as_half((unsigned short)(i & 1 ? w >> 16 : w & 0xFFFFu)));
}
template <> __device__ __forceinline__ float Raw<__half, 4>::get(int i) const { return f16_at(w[i >> 1], i); }
template <> __device__ __forceinline__ float Raw<__half, 2>::get(int i) const { return f16_at(w[0], i); }

// The byte mask of the V word with tokens 16 w + 2 c + {0, 1, 8, 9}, from a mask of the block's tokens.
__device__ __forceinline__ uint32_t v_word_mask(uint32_t tokens, int c, int w) {
  const uint32_t t = tokens >> (16 * w + 2 * c);
  return (t & 1 ? 0xFFu : 0u) | (t & 2 ? 0xFF00u : 0u) | (t & 0x100 ? 0xFF0000u : 0u) | (t & 0x200 ? 0xFF000000u : 0u);
}

// Runs among 32 consecutive entries base .. of a slot list (of which `chunk`
// may start one): entries whose slots follow one another in a block.
struct Runs {
  int s0, s1;                      // slot of entry base + lane, base + 32 + lane; -1: outside the pool or the list
  uint32_t starts;                 // entries that start a run
  __device__ __forceinline__ Runs(const int32_t* slot, int n, int slots, int base, int chunk) {
    const int lane = threadIdx.x & 31;
    auto at = [&](int i) {
      const int s = i >= 0 && i < n ? slot[i] : -1;
      return s < slots ? s : -1;
    };
    s0 = at(base + lane);
    s1 = at(base + 32 + lane);
    const int first_before = lane == 0 ? at(base - 1) : 0;
    const int up = __shfl_up_sync(0xffffffffu, s0, 1);
    const int before = lane == 0 ? first_before : up;
    starts = __ballot_sync(0xffffffffu, lane < chunk && s0 >= 0 && !(before >= 0 && s0 == before + 1 && (s0 & 31)));
  }
  // The run that starts at entry `first`: its slot and length.
  __device__ __forceinline__ int run(int first, int* len) const {
    const int lane = threadIdx.x & 31;
    const int s = __shfl_sync(0xffffffffu, s0, first);
    const uint32_t e0 = __ballot_sync(0xffffffffu, s0 == s + (lane - first) && (s0 >> 5) == (s >> 5));
    const uint32_t e1 = __ballot_sync(0xffffffffu, s1 == s + (lane + 32 - first) && (s1 >> 5) == (s >> 5));
    const uint64_t e = ((uint64_t)e1 << 32 | e0) >> first;
    *len = min(__ffsll((long long)~e) - 1, 32);
    return s;
  }
};

// A warp: the runs that start in `chunk` consecutive rows, of one head, of K
// (z = 0) or V (z = 1).  A lane has D / 32 dimensions of every row.  A long
// run is read once into registers, all rows in flight; a K row leaves as 4
// bytes a lane, and V needs no exchange between lanes, since the 16-byte pieces of
// its layout (two dimensions, eight tokens) each lie with one lane.  A decode step's runs
// are one row each: V's bytes go out one by one, less than a block's way in and out.
// Bound by HBM, two or four bytes in for one out: 14.6k bf16 rows of 8
// heads of 128 in 20.1 us, 4.5 TB/s, 68 % of a copy, fp32 rows in 32.2 us, 71 % (of
// the rest most is the last wave of these 1824 CTAs, 3.1 of four an SM); 32
// fp32 rows of 32 heads in 5.2 us, a launch and two dependent reads.
template <typename T, int D>
__global__ void __launch_bounds__(kCopyWarps * 32)
    kv_append_kernel(KvView c, const T* __restrict__ k, long k_stride, const T* __restrict__ v, long v_stride,
                     const int32_t* __restrict__ slot, int n, int chunk) {
  constexpr int V = D / 32;        // dimensions a lane
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int base = (blockIdx.x * kCopyWarps + warp) * chunk, head = blockIdx.y;
  if (base >= n) return;
  const bool is_v = blockIdx.z != 0;
  const T* src = (is_v ? v : k) + (long)head * D + lane * V;
  const long stride = is_v ? v_stride : k_stride;
  int8_t* data = is_v ? c.v : c.k;
  uint8_t* scales = is_v ? c.vs : c.ks;
  const Runs runs(slot, n, c.n_pages * c.page, base, chunk);

  for (uint32_t left = runs.starts; left; left &= left - 1) {
    int len;
    const int first = __ffs((int)left) - 1, s0 = runs.run(first, &len), o = s0 & 31;
    const long blk = kv_block(c, s0 / c.page, head, (s0 % c.page) >> 5);
    uint8_t* dst = reinterpret_cast<uint8_t*>(data) + blk * (32 * D);
    const int was = o ? scales[blk] : 0;
    const T* rows = src + (long)(base + first) * stride;
    if (len < kLongRun) {
      uint32_t top = 0;
      Raw<T, V> x;
      for (int r = 0; r < len; ++r) {
        x.load(rows + (long)r * stride);
        top = x.top(top);
      }
      top = __reduce_max_sync(0xffffffffu, f32_bits<T>(top));
      const int byte = max(scale_byte(top), was);
      if (o && byte > was && byte != 255) {
        const float down = step_down(was, byte);
#pragma unroll
        for (int u = 0; u < 2 * D / 32; ++u) {
          uint4* w = reinterpret_cast<uint4*>(dst) + u * 32 + lane;
          *w = reround16(*w, down);
        }
        __syncwarp();
      }
      const float inv = byte == 255 ? 0.0f : pow2_exact(127 - byte);
      for (int r = 0; r < len; ++r) {
        if (len > 1) x.load(rows + (long)r * stride);
        uint32_t w = 0;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const uint32_t q = byte == 255 ? 0u : quant_bits(x.get(e), inv) & 0xFF;
          if (is_v) dst[v_offset(o + r, lane * V + e)] = (uint8_t)q;
          w |= q << (8 * e);
        }
        if (!is_v) {
          if (V == 4) *reinterpret_cast<uint32_t*>(dst + (o + r) * D + lane * 4) = w;
          else *reinterpret_cast<uint16_t*>(dst + (o + r) * D + lane * 2) = (uint16_t)w;
        }
      }
      if (lane == 0) scales[blk] = (uint8_t)byte;
      continue;
    }

    // x[t]: the row of the block's token t
    Raw<T, V> x[32];
#pragma unroll
    for (int t = 0; t < 32; ++t) {
      if (t >= o && t < o + len) x[t].load(rows + (long)(t - o) * stride);
      else x[t].clear();
    }
    uint32_t top = 0;
#pragma unroll
    for (int t = 0; t < 32; ++t) top = x[t].top(top);
    top = __reduce_max_sync(0xffffffffu, f32_bits<T>(top));
    const int byte = max(scale_byte(top), was);
    const bool grew = o && byte > was && byte != 255;
    const float down = grew ? step_down(was, byte) : 1.0f;
    const float inv = byte == 255 ? 0.0f : pow2_exact(127 - byte);
    const uint32_t tokens = (len == 32 ? 0xffffffffu : (1u << len) - 1) << o;
    if (byte == 255) {
#pragma unroll
      for (int t = 0; t < 32; ++t) x[t].clear();
    }
    if (!is_v) {
#pragma unroll
      for (int t = 0; t < 32; ++t) {
        uint32_t w = 0;
        if (V == 4) {
          const uint32_t lo = __byte_perm(quant_bits(x[t].get(0), inv), quant_bits(x[t].get(1), inv), 0x0040);
          const uint32_t hi = __byte_perm(quant_bits(x[t].get(2 % V), inv), quant_bits(x[t].get(3 % V), inv), 0x0040);
          w = __byte_perm(lo, hi, 0x5410);
          uint32_t* to = reinterpret_cast<uint32_t*>(dst + t * D + lane * 4);
          if (tokens >> t & 1) *to = w;
          else if (grew) *to = reround4(*to, down);
        } else {
          w = __byte_perm(quant_bits(x[t].get(0), inv), quant_bits(x[t].get(1), inv), 0x0040);
          uint16_t* to = reinterpret_cast<uint16_t*>(dst + t * D + lane * 2);
          if (tokens >> t & 1) *to = (uint16_t)w;
          else if (grew) *to = (uint16_t)reround4(*to, down);
        }
      }
    } else {
#pragma unroll
      for (int pr = 0; pr < V / 2; ++pr)
#pragma unroll
        for (int cc = 0; cc < 4; ++cc) {
          uint32_t w[4];           // dimension 2 pr: tokens of words 0, 1; then 2 pr + 1
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int t0 = 16 * (e & 1) + 2 * cc, d = 2 * pr + (e >> 1);
            const uint32_t lo = __byte_perm(quant_bits(x[t0].get(d), inv), quant_bits(x[t0 + 1].get(d), inv), 0x0040);
            const uint32_t hi = __byte_perm(quant_bits(x[t0 + 8].get(d), inv), quant_bits(x[t0 + 9].get(d), inv), 0x0040);
            w[e] = __byte_perm(lo, hi, 0x5410);
          }
          uint4* to = reinterpret_cast<uint4*>(dst) + (lane * (V / 2) + pr) * 4 + cc;
          if (o) {                 // the block's other tokens stay
            uint4 old = *to;
            if (grew) old = reround16(old, down);
            const uint32_t m0 = v_word_mask(tokens, cc, 0), m1 = v_word_mask(tokens, cc, 1);
            w[0] = (w[0] & m0) | (old.x & ~m0);
            w[1] = (w[1] & m1) | (old.y & ~m1);
            w[2] = (w[2] & m0) | (old.z & ~m0);
            w[3] = (w[3] & m1) | (old.w & ~m1);
          }
          *to = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
    if (lane == 0) scales[blk] = (uint8_t)byte;
  }
}

// ------------------------------------------------------------------ read --

// Byte b of a word of int8 as a float: 2^23 + 128 + x from its bits, less 2^23 + 128.
__device__ __forceinline__ float int8_value(uint32_t flipped, int b) {   // flipped: w ^ 0x80808080
  return __uint_as_float(__byte_perm(flipped, 0x4B000000u, 0x7540 | b)) - 8388736.0f;
}

// N consecutive values, N * sizeof(T) bytes aligned.
__device__ __forceinline__ void put2(float* p, float a, float b) { *reinterpret_cast<float2*>(p) = make_float2(a, b); }
__device__ __forceinline__ void put2(__nv_bfloat16* p, float a, float b) {
  *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(a, b);
}
__device__ __forceinline__ void put2(__half* p, float a, float b) {
  *reinterpret_cast<__half2*>(p) = __floats2half2_rn(a, b);
}

// A warp: `chunk` consecutive entries, of one head, of K or V.  K rows are read
// four at a time.  V is read a run at a time, whole blocks in 16-byte pieces: a
// lane has two dimensions of eight tokens, and four lanes' stores reach
// four rows in whole sectors.  Bound by HBM: 14.7k rows of 8 heads to bf16 in
// 20.2 us, 4.5 TB/s; 444 rows of 32 heads to bf16 in 5.8 us.
template <typename T, int D>
__global__ void __launch_bounds__(kCopyWarps * 32)
    kv_read_kernel(KvView c, const int32_t* __restrict__ slot, int n, int chunk, T* __restrict__ k_out,
                   T* __restrict__ v_out) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int base = (blockIdx.x * kCopyWarps + warp) * chunk, head = blockIdx.y;
  if (base >= n) return;
  const bool is_v = blockIdx.z != 0;
  const Runs runs(slot, n, c.n_pages * c.page, base, chunk);
  const int count = min(chunk, n - base);
  const long row = (long)c.heads * D;
  T* out = (is_v ? v_out : k_out) + (long)base * row + (long)head * D;
  // entries outside the pool
  for (uint32_t z = __ballot_sync(0xffffffffu, lane < count && runs.s0 < 0); z; z &= z - 1) {
    T* to = out + (long)(__ffs((int)z) - 1) * row;
    for (int d = 2 * lane; d < D; d += 64) put2(to + d, 0.0f, 0.0f);
  }
  if (!is_v) {
    constexpr int kLanes = D / 16, kRows = 32 / kLanes;    // 16 dimensions a lane
    for (int i0 = 0; i0 < count; i0 += kRows) {
      const int i = i0 + lane / kLanes;
      const int s = __shfl_sync(0xffffffffu, runs.s0, i & 31);
      if (i >= count || s < 0) continue;
      const long blk = kv_block(c, s / c.page, head, (s % c.page) >> 5);
      const uint4 w = __ldg(reinterpret_cast<const uint4*>(c.k + blk * (32 * D) + (s & 31) * D) + lane % kLanes);
      const float sc = e8m0_to_float(c.ks[blk]);
      const uint32_t q[4] = {w.x, w.y, w.z, w.w};
      T* to = out + (long)i * row + (lane % kLanes) * 16;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float y[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) y[b] = int8_value(q[e] ^ 0x80808080u, b) * sc;
        store4(to + 4 * e, y);
      }
    }
    return;
  }
  // a run may have started before this warp's entries: its first entry here counts as a start
  const int s_first = __shfl_sync(0xffffffffu, runs.s0, 0);
  uint32_t left = runs.starts | (s_first >= 0 ? 1u : 0u);
  for (; left; left &= left - 1) {
    int len;
    const int first = __ffs((int)left) - 1, s0 = runs.run(first, &len), o = s0 & 31;
    len = min(len, count - first);
    const long blk = kv_block(c, s0 / c.page, head, (s0 % c.page) >> 5);
    const uint4* src = reinterpret_cast<const uint4*>(c.v + blk * (32 * D));
    const float sc = e8m0_to_float(c.vs[blk]);
    const int cc = lane & 3;
    uint4 w[D / 16];
#pragma unroll
    for (int u = 0; u < D / 16; ++u) {
      w[u] = __ldg(src + u * 32 + lane);
      w[u].x ^= 0x80808080u; w[u].y ^= 0x80808080u; w[u].z ^= 0x80808080u; w[u].w ^= 0x80808080u;
    }
#pragma unroll
    for (int jb = 0; jb < 8; ++jb) {
      const int r = (jb >> 1) * 8 + 2 * cc + (jb & 1) - o;   // the token's entry in the run
      if (r < 0 || r >= len) continue;
      T* to = out + (long)(first + r) * row + 2 * (lane >> 2);
#pragma unroll
      for (int u = 0; u < D / 16; ++u) {
        const uint32_t a = jb < 4 ? w[u].x : w[u].y, b = jb < 4 ? w[u].z : w[u].w;
        put2(to + u * 16, int8_value(a, jb & 3) * sc, int8_value(b, jb & 3) * sc);
      }
    }
  }
}

// Rows a warp looks for runs in: 32 (a prompt's warp then has a block or two),
// fewer while that many warps would leave the SMs without 16 each: a decode step's runs
// are one row, and a warp takes its runs one after another (32 rows x 32
// heads: 9.0 us with 8 rows a warp, 5.0 with one).
int rows_a_warp(const KvView& c, int n) {
  const long units = 2l * n * c.heads, enough = 148l * 16;
  return units / 32 >= enough ? 32 : units / 8 >= enough ? 8 : 1;
}

template <typename T>
cudaError_t launch_append(const KvView& c, const void* k, long k_stride, const void* v, long v_stride,
                          const int32_t* slot, int n, cudaStream_t st) {
  const int chunk = rows_a_warp(c, n), per = chunk * kCopyWarps;
  const dim3 grid((unsigned)((n + per - 1) / per), (unsigned)c.heads, 2);
  if (c.dim == 64)
    kv_append_kernel<T, 64><<<grid, kCopyWarps * 32, 0, st>>>(c, static_cast<const T*>(k), k_stride,
                                                              static_cast<const T*>(v), v_stride, slot, n, chunk);
  else
    kv_append_kernel<T, 128><<<grid, kCopyWarps * 32, 0, st>>>(c, static_cast<const T*>(k), k_stride,
                                                               static_cast<const T*>(v), v_stride, slot, n, chunk);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_read(const KvView& c, const int32_t* slot, int n, void* k, void* v, cudaStream_t st) {
  const int chunk = rows_a_warp(c, n), per = chunk * kCopyWarps;
  const dim3 grid((unsigned)((n + per - 1) / per), (unsigned)c.heads, 2);
  if (c.dim == 64)
    kv_read_kernel<T, 64><<<grid, kCopyWarps * 32, 0, st>>>(c, slot, n, chunk, static_cast<T*>(k), static_cast<T*>(v));
  else
    kv_read_kernel<T, 128><<<grid, kCopyWarps * 32, 0, st>>>(c, slot, n, chunk, static_cast<T*>(k), static_cast<T*>(v));
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
  // a thread a new row (or request) up to one CTA an SM, in CTAs of 256 while
  // 16 of them will do; up to 256 rows are one CTA's
  const size_t most = n_tokens > n_req ? n_tokens : n_req;
  const int threads = most <= 4096 ? 256 : 1024;
  size_t ctas = (most + threads - 1) / threads;
  if (ctas > (size_t)ws.sms) ctas = (size_t)ws.sms;
  const size_t smem = (3 * n_req + 2) * sizeof(int);
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
  return mxq_kv_append_strided(c, cache, dtype, k, row_stride, v, row_stride, slot, n);
}

int mxq_kv_append_strided(mxq_ctx c, const mxq_kv_cache* cache, int dtype, const void* k, size_t k_stride, const void* v,
                          size_t v_stride, const int32_t* slot, size_t n) {
  if (!c) return bad(nullptr, "null context");
  KvView kv;
  if (const char* msg = kv_view(cache, &kv)) return bad(c, msg);
  const size_t es = dtype_bytes(dtype);
  if (!es) return bad(c, "kv append: unknown row type");
  if (n == 0) return MXQ_OK;
  if (!k || !v || !slot) return bad(c, "kv append: null pointer");
  if (n > (1u << 30)) return bad(c, "kv append: too many rows");
  const size_t row = (size_t)kv.heads * kv.dim;
  if (k_stride < row || v_stride < row) return bad(c, "kv append: rows overlap");
  if (!aligned16(k) || !aligned16(v) || k_stride * es % 16 || v_stride * es % 16)
    return bad(c, "kv append: rows must start on 16-byte boundaries");
  ServeDevice g(ctx_device(c));
  const cudaStream_t st = ctx_stream(c);
  const cudaError_t e =
      dtype == MXQ_DT_F32 ? launch_append<float>(kv, k, (long)k_stride, v, (long)v_stride, slot, (int)n, st)
      : dtype == MXQ_DT_BF16 ? launch_append<__nv_bfloat16>(kv, k, (long)k_stride, v, (long)v_stride, slot, (int)n, st)
                             : launch_append<__half>(kv, k, (long)k_stride, v, (long)v_stride, slot, (int)n, st);
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
