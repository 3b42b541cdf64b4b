// mxq_logprob.cu -- log probabilities of given tokens with entropy and top
// alternatives, and the gradient to the logits (the rollout head of
// PPOTrainer::update_step, training/ppo_trainer.cpp:64-66 and :77, for a
// vocabulary, where the actions are token ids and not rows of weights).
//
// With M = max_j x_j, s = sum_j exp(x_j - M) and u = sum_j exp(x_j - M)(x_j - M):
//   lse = M + log s,  logp = (x_t - M) - log s,  entropy = log s - u / s.
// Forward: one pass over the row; every thread keeps (M, s, u) of what it has
// read and rescales when its M rises, so the row is read from memory once.
// A pass has nothing to reuse, and HBM bounds fp32 rows and the gradient: 8192
// rows of 32000 fp32 logits with 5 alternatives take 167 to 170 us launch after
// launch, 175 with cold caches, 6.1 TB/s, 92 % of a copy; the gradient of 4096 x
// 32000 bf16 82 us, 6.4 TB/s, of fp32 157 us.  16-bit rows do the same work
// for each logit in half the bytes and are bound by its instructions: 8192 x 32000
// bf16 158 us, twice their bytes' time.  One row of 32000 is bound by latency: 5.9 us.
#include "mxq_serve.cuh"

namespace mxq {

namespace {

constexpr int kMaxSlices = 8;      // CTAs a row (a portable cluster)
constexpr int kCandidates = 1024;

// Order of the top alternatives as one integer: descending logit (NaN above
// all, -0 equal to 0), then ascending id.  0 is below every real entry.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0xFFFFFFFFu;
  const uint32_t b = __float_as_uint(x + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {   // of an entry; of 0, a NaN
  if (k == 0xFFFFFFFFu) return __int_as_float(0x7fc00000);
  return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}
__device__ __forceinline__ uint64_t order_entry(float x, int id) {
  return (uint64_t)order_key(x) << 32 | (0xFFFFFFFFu - (uint32_t)id);
}

// What a thread, warp or CTA knows of the row so far.
struct Stat {
  float m, s, u;
};
__device__ __forceinline__ float floor_max(float m) { return fmaxf(m, -3.402823466e38f); }
// A difference to the maximum, finite: beyond -1000 its exp is 0 either way,
// and 0 times it must be 0 (a mask of the type's lowest value, -inf).
__device__ __forceinline__ float drop(float d) { return fmaxf(d, -1000.0f); }
__device__ __forceinline__ Stat merge(const Stat& a, const Stat& b) {
  const float m = fmaxf(a.m, b.m), f = floor_max(m);
  const float da = drop(floor_max(a.m) - f), db = drop(floor_max(b.m) - f);
  const float ca = ex2(da * kLog2e), cb = ex2(db * kLog2e);
  return {m, a.s * ca + b.s * cb, ca * (a.u + a.s * da) + cb * (b.u + b.s * db)};
}
__device__ __forceinline__ Stat shfl_xor(const Stat& a, int o) {
  return {__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o),
          __shfl_xor_sync(0xffffffffu, a.u, o)};
}

// Where a thread's largest value is: its batch, and the largest of its other batches.
struct Largest {
  int at;                          // the batch's first vector, -1: the ends of the row
  float other;
};

// N values, the batch `at`, into a thread's statistics.
template <int N>
__device__ __forceinline__ void add_values(Stat& t, Largest& g, int at, const float (&x)[N]) {
  float top = x[0];
#pragma unroll
  for (int i = 1; i < N; ++i) top = fmaxf(top, x[i]);
  g.other = fmaxf(g.other, fminf(top, t.m));
  if (top > t.m) {
    g.at = at;
    const float f = floor_max(top), d = drop(floor_max(t.m) - f), c = ex2(d * kLog2e);
    t.u = c * (t.u + t.s * d);
    t.s *= c;
    t.m = top;
  }
  const float f = floor_max(t.m);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float d = x[i] - f;
    const float e = ex2(d * kLog2e);
    t.s += e;
    t.u = fmaf(e, drop(d), t.u);
  }
}

// 16 bytes of a row as values.
template <typename T> struct Vec { static constexpr int kN = 16 / (int)sizeof(T); };
template <typename T>
__device__ __forceinline__ void unpack16(const uint4& w, float* v);
template <> __device__ __forceinline__ void unpack16<float>(const uint4& w, float* v) {
  v[0] = __uint_as_float(w.x); v[1] = __uint_as_float(w.y); v[2] = __uint_as_float(w.z); v[3] = __uint_as_float(w.w);
}
template <> __device__ __forceinline__ void unpack16<__nv_bfloat16>(const uint4& w, float* v) {
  const uint32_t a[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(a[i] << 16);
    v[2 * i + 1] = __uint_as_float(a[i] & 0xFFFF0000u);
  }
}
template <> __device__ __forceinline__ void unpack16<__half>(const uint4& w, float* v) {
  const uint32_t a[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&a[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

// A row cut at 16-byte boundaries: `head` elements before the first, nv whole
// vectors, `tail` elements after the last.  Slice `rank` of `slices` takes the
// vectors rank * THREADS + tid, + slices * THREADS, ...; slice 0 the ends too.
template <typename T>
struct RowView {
  const T* x;
  const uint4* body;
  int head, nv, tail, vocab;
  __device__ __forceinline__ RowView(const T* row, int n) : x(row), vocab(n) {
    const int mis = (int)((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T));
    head = mis ? Vec<T>::kN - mis : 0;
    if (head > n) head = n;
    nv = (n - head) / Vec<T>::kN;
    tail = n - head - nv * Vec<T>::kN;
    body = reinterpret_cast<const uint4*>(row + head);
  }
  // place of the i-th element outside the vectors
  __device__ __forceinline__ int end(int i) const { return i < head ? i : vocab - tail + (i - head); }
  // f(value, id) for every element of this thread
  template <int THREADS, typename F>
  __device__ __forceinline__ void each(int rank, int slices, F f) const {
    const int tid = threadIdx.x;
    if (rank == 0)
      for (int i = tid; i < head + tail; i += THREADS) f(to_f32(x[end(i)]), end(i));
    for (int i = rank * THREADS + tid; i < nv; i += slices * THREADS) {
      float v[Vec<T>::kN];
      unpack16<T>(__ldg(body + i), v);
#pragma unroll
      for (int e = 0; e < Vec<T>::kN; ++e) f(v[e], head + i * Vec<T>::kN + e);
    }
  }
};

struct LogprobArgs {
  const void* logits;
  long stride;
  int rows, vocab, k, slices;
  const int32_t* target;
  float *logp, *entropy, *lse, *top_logp;
  int32_t* top_ids;
};

template <int THREADS>
struct LogprobShared {
  Stat warp[THREADS / 32];
  Stat all;                        // this slice's statistics
  uint32_t group[32];
  uint64_t cand[kCandidates];
  uint64_t best[MXQ_TOPK_MAX];     // this slice's top entries, in order
  uint64_t pick[THREADS / 32];
  int count;
  uint32_t threshold;
};

// Entries in order: place = how many are above.  Entries differ (the id is
// part of them), so places do too.
__device__ __forceinline__ void place_entries(const uint64_t* in, int n, int k, uint64_t* out, int threads) {
  for (int i = threadIdx.x; i < n; i += threads) {
    const uint64_t e = in[i];
    if (!e) continue;
    int above = 0;
    for (int j = 0; j < n; ++j) above += in[j] > e;
    if (above < k) out[above] = e;
  }
}

// The same for `lists` ordered lists of MXQ_TOPK_MAX entries (0 beyond their
// ends): an entry's place is its own in its list and, from each other list, the
// entries above it.
__device__ __forceinline__ void merge_entries(const uint64_t* in, int lists, int k, uint64_t* out, int threads) {
  static_assert(MXQ_TOPK_MAX == 32, "five steps");
  for (int i = threadIdx.x; i < lists * MXQ_TOPK_MAX; i += threads) {
    const uint64_t e = in[i];
    if (!e) continue;
    int above = i % MXQ_TOPK_MAX;
    for (int l = 0; l < lists; ++l) {
      if (l == i / MXQ_TOPK_MAX) continue;
      const uint64_t* p = in + l * MXQ_TOPK_MAX;
      int n = 0;                   // entries of the list known to be above
#pragma unroll
      for (int step = 16; step > 0; step >>= 1)
        if (p[n + step - 1] > e) n += step;
      above += n + (p[n] > e);
    }
    if (above < k) out[above] = e;
  }
}

// One row, `slices` CTAs (a cluster when there are several: few rows leave
// SMs idle, and a row is long).  The top alternatives need no second pass
// over the row: every group of THREADS / 32 threads knows its largest logit, so the
// k-th largest of these 32 is a bound that at least k logits reach.  A thread whose
// own maximum reaches it reads the batch of 8 that has it again, and all of its part
// only where another of its batches reaches the bound too.
template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS) token_logprobs_kernel(LogprobArgs a) {
  __shared__ LogprobShared<THREADS> sh;
  // vectors a thread has on the way: 8 where many rows share an SM (8192 rows: 167 us,
  // with 4 173, with 12 186), 4 where one row's latency counts (5.9 us, with 8 6.3)
  constexpr int kN = Vec<T>::kN, kAhead = THREADS == 256 ? 8 : 4;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int slices = a.slices, rank = slices > 1 ? (int)cluster_ctarank() : 0;
  const long row = blockIdx.x / slices;
  const RowView<T> rv(static_cast<const T*>(a.logits) + row * a.stride, a.vocab);

  Stat t{neg_inf(), 0.0f, 0.0f};
  Largest g{-1, t.m};
  bool any = false;
  if (rank == 0) {
    for (int i = tid; i < rv.head + rv.tail; i += THREADS) {
      const float v[1] = {to_f32(rv.x[rv.end(i)])};
      add_values(t, g, -1, v);
      any = true;
    }
  }
  // kAhead vectors on the way while the last ones are added, 8 values at a time
  constexpr int kPair = 8 / kN;
  const int step = slices * THREADS;
  uint4 w[kAhead];
  int i = rank * THREADS + tid;
  any = any || i < rv.nv;
#pragma unroll
  for (int u = 0; u < kAhead; ++u)
    if (i + u * step < rv.nv) w[u] = __ldcs(rv.body + i + u * step);
  for (; i + (kAhead - 1) * step < rv.nv; i += kAhead * step) {
#pragma unroll
    for (int u = 0; u < kAhead; u += kPair) {
      float v[8];
#pragma unroll
      for (int q = 0; q < kPair; ++q) {
        unpack16<T>(w[u + q], v + q * kN);
        const int nx = i + (kAhead + u + q) * step;
        if (nx < rv.nv) w[u + q] = __ldcs(rv.body + nx);
      }
      add_values(t, g, i + u * step, v);
    }
  }
#pragma unroll
  for (int u = 0; u < kAhead; ++u)
    if (i + u * step < rv.nv) {
      float v[kN];
      unpack16<T>(w[u], v);
      add_values(t, g, i + u * step, v);
    }
  const uint32_t mine = any ? order_key(t.m) : 0u;

  // the slice's statistics
  Stat r = t;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) r = merge(r, shfl_xor(r, o));
  if (lane == 0) sh.warp[warp] = r;
  if (a.k > 0) {
    uint32_t top = mine;
    constexpr int kGroup = THREADS / 32;
#pragma unroll
    for (int o = kGroup / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (tid % kGroup == 0) sh.group[tid / kGroup] = top;
  }
  if (tid == 0) sh.count = 0;
  if (tid < MXQ_TOPK_MAX) sh.best[tid] = 0;
  __syncthreads();
  if (warp == 0) {
    Stat w = lane < THREADS / 32 ? sh.warp[lane] : Stat{neg_inf(), 0.0f, 0.0f};
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) w = merge(w, shfl_xor(w, o));
    if (lane == 0) sh.all = w;
    if (a.k > 0) {
      const uint32_t g = sh.group[lane];
      int above = 0;
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        const uint32_t o = __shfl_sync(0xffffffffu, g, j);
        above += o > g || (o == g && j < lane);
      }
      if (above == a.k - 1) sh.threshold = g;
    }
  }
  __syncthreads();

  if (a.k > 0) {
    const uint32_t least = sh.threshold;
    const bool odd = !(sh.all.s == sh.all.s);     // a NaN or +inf among them: the maxima are not to be trusted
    if (!odd) {
      const float bound = key_value(least);       // least 0: a group without logits, every logit counts
      auto test = [&](float x, int id) {
        if (least == 0u || x >= bound) {
          const int at = atomicAdd(&sh.count, 1);
          if (at < kCandidates) sh.cand[at] = order_entry(x, id);
        }
      };
      const bool reaches = any && mine >= least;
      const bool many = reaches && (least == 0u || g.other >= bound);
      if (reaches && !many) {
        // one batch: its second vector is a batch of its own near the row's end, and below the bound
        if (g.at < 0)
          test(to_f32(rv.x[rv.end(tid)]), rv.end(tid));
        else
          for (int q = 0; q < kPair && g.at + q * step < rv.nv; ++q) {
            float v[kN];
            unpack16<T>(__ldg(rv.body + g.at + q * step), v);
#pragma unroll
            for (int e = 0; e < kN; ++e) test(v[e], rv.head + (g.at + q * step) * kN + e);
          }
      }
      // several: a warp looks through the part of each such lane in turn, a vector a lane
      for (uint32_t left = __ballot_sync(0xffffffffu, many); left; left &= left - 1) {
        const int who = warp * 32 + __ffs((int)left) - 1;
        if (rank == 0 && lane == 0 && who < rv.head + rv.tail) test(to_f32(rv.x[rv.end(who)]), rv.end(who));
        for (int j = rank * THREADS + who + lane * step; j < rv.nv; j += 32 * step) {
          float v[kN];
          unpack16<T>(__ldg(rv.body + j), v);
#pragma unroll
          for (int e = 0; e < kN; ++e) test(v[e], rv.head + j * kN + e);
        }
      }
    }
    __syncthreads();
    const int n = sh.count;
    if (!odd && n <= kCandidates) {
      place_entries(sh.cand, n, a.k, sh.best, THREADS);
    } else {
      // many equal logits, or NaN: one entry at a time, the largest below the last
      uint64_t last = 0;
      for (int j = 0; j < a.k; ++j) {
        uint64_t e = 0;
        rv.template each<THREADS>(rank, slices, [&](float x, int id) {
          const uint64_t c = order_entry(x, id);
          if ((j == 0 || c < last) && c > e) e = c;
        });
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const uint64_t c = __shfl_xor_sync(0xffffffffu, e, o);
          e = c > e ? c : e;
        }
        if (lane == 0) sh.pick[warp] = e;
        __syncthreads();
        for (int w = 0; w < THREADS / 32; ++w) e = sh.pick[w] > e ? sh.pick[w] : e;
        last = e;
        if (tid == 0) sh.best[j] = e;
        __syncthreads();
        if (!e) break;                            // the slice has no more (uniform)
      }
    }
    __syncthreads();
  }

  if (slices > 1) cluster_sync_all();
  if (rank == 0) {
    Stat all = sh.all;
    if (slices > 1) {
      const uint32_t base = smem_u32(&sh.all);
      for (int s = 1; s < slices; ++s) {
        const uint32_t at = mapa_shared(base, s);
        Stat o;
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(o.m) : "r"(at) : "memory");
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(o.s) : "r"(at + 4) : "memory");
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(o.u) : "r"(at + 8) : "memory");
        all = merge(all, o);
      }
      if (a.k > 0) {
        for (int e = tid; e < slices * MXQ_TOPK_MAX; e += THREADS) {
          const uint32_t at = mapa_shared(smem_u32(&sh.best[e % MXQ_TOPK_MAX]), e / MXQ_TOPK_MAX);
          uint64_t v;
          asm volatile("ld.shared::cluster.b64 %0, [%1];" : "=l"(v) : "r"(at) : "memory");
          sh.cand[e] = v;
        }
        __syncthreads();
        merge_entries(sh.cand, slices, a.k, sh.best, THREADS);
        __syncthreads();
      }
    }
    const float logs = logf(all.s);               // -inf where nothing is left
    const bool empty = all.s == 0.0f;
    if (tid == 0) {
      const int tgt = a.target[row];
      float lp = 0.0f;
      if (tgt >= 0 && tgt < a.vocab) lp = empty ? neg_inf() : (to_f32(rv.x[tgt]) - all.m) - logs;
      if (a.logp) a.logp[row] = lp;
      if (a.lse) a.lse[row] = empty ? neg_inf() : all.m + logs;
      if (a.entropy) a.entropy[row] = empty ? 0.0f : logs - all.u / all.s;
    }
    if (tid < a.k) {
      const uint64_t e = sh.best[tid];
      const float x = key_value((uint32_t)(e >> 32));
      a.top_logp[row * a.k + tid] = empty ? neg_inf() : (x - all.m) - logs;
      a.top_ids[row * a.k + tid] = (int32_t)(0xFFFFFFFFu - (uint32_t)e);
    }
  }
  if (slices > 1) cluster_sync_all();             // nobody's shared memory goes before the leader has read it
}

// -------------------------------------------------------------- gradient --

struct LogprobGradArgs {
  const void* logits;
  void* grad;
  long stride, grad_stride;
  int rows, vocab, per_row;        // CTAs a row
  const int32_t* target;
  const float *lse, *entropy, *dlogp, *dentropy;
};

template <typename T>
__device__ __forceinline__ void store16(T* p, const float* v);
template <> __device__ __forceinline__ void store16(float* p, const float* v) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
template <> __device__ __forceinline__ void store16(__nv_bfloat16* p, const float* v) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&b);
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
template <> __device__ __forceinline__ void store16(__half* p, const float* v) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 b = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&b);
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

constexpr int kGradThreads = 256;
// vectors a thread has on the way, and times that, a CTA (4096 rows of 32000 bf16:
// 82.5 us with 2 and 2, 85.2 with 4 and 2, 88.2 with 4 and 4)
constexpr int kGradBatch = 2;
constexpr int kGradLoops = 2;

// dx_j = dlogp (1[j = t] - p_j) - dentropy p_j (log p_j + H): 16-byte stores at
// the gradient's alignment, the logits in 16 bytes where they share it.  The
// target's element is the only one with a second term: the thread that has
// it adds it there.
template <typename T>
__global__ void __launch_bounds__(kGradThreads) token_logprobs_grad_kernel(LogprobGradArgs a) {
  constexpr int kN = Vec<T>::kN;
  const long row = blockIdx.x / a.per_row;
  const int part = blockIdx.x % a.per_row, tid = threadIdx.x;
  const T* x = static_cast<const T*>(a.logits) + row * a.stride;
  T* g = static_cast<T*>(a.grad) + row * a.grad_stride;
  const int mis = (int)((reinterpret_cast<uintptr_t>(g) & 15u) / sizeof(T));
  const int head = min(mis ? kN - mis : 0, a.vocab);
  const int nv = (a.vocab - head) / kN;
  const bool same = (reinterpret_cast<uintptr_t>(x + head) & 15u) == 0;
  const int per_cta = kGradThreads * kGradBatch * kGradLoops;
  int first = part * per_cta + tid;
  const int end = min(nv, (part + 1) * per_cta);
  uint4 w[kGradBatch];
  auto load_one = [&](int i, uint4& to) {
    const T* from = x + head + (long)i * kN;
    if (same) {
      to = __ldcs(reinterpret_cast<const uint4*>(from));
    } else if (sizeof(T) == 4) {
      const uint32_t* p = reinterpret_cast<const uint32_t*>(from);
      to = make_uint4(p[0], p[1], p[2], p[3]);
    } else {
      const uint16_t* p = reinterpret_cast<const uint16_t*>(from);
      auto two = [&](int e) { return (uint32_t)p[e] | (uint32_t)p[e + 1] << 16; };
      to = make_uint4(two(0), two(2), two(4 % kN), two(6 % kN));
    }
  };
#pragma unroll
  for (int u = 0; u < kGradBatch; ++u)
    if (first + u * kGradThreads < end) load_one(first + u * kGradThreads, w[u]);
  const float lse = a.lse[row], h = a.entropy ? a.entropy[row] : 0.0f;
  // nothing but banned tokens, by -inf or by the lowest value of fp32 or bf16: log p
  // cannot be had from lse there, and no token is to be pushed anywhere
  const bool empty = lse < -1e30f;
  const int tgt = a.target[row];
  const float dl = a.dlogp && tgt >= 0 && tgt < a.vocab && !empty ? a.dlogp[row] : 0.0f;
  const float de = a.dentropy && !empty ? a.dentropy[row] : 0.0f;
  const float c = -fmaf(de, h, dl);
  auto one = [&](float y) {
    const float lp = empty ? -1000.0f : y - lse;
    // p (c - de log p), with a finite log p where p is 0
    return ex2(lp * kLog2e) * fmaf(-de, drop(lp), c);
  };
  if (part == 0) {
    for (int i = tid; i < head; i += kGradThreads) {
      const float r = one(to_f32(x[i]));
      g[i] = from_f32<T>(i == tgt ? dl + r : r);
    }
    for (int i = head + nv * kN + tid; i < a.vocab; i += kGradThreads) {
      const float r = one(to_f32(x[i]));
      g[i] = from_f32<T>(i == tgt ? dl + r : r);
    }
  }
  const int tv = tgt >= head ? (tgt - head) / kN : -1;   // the target's vector, and its element
  const int te = tv >= 0 ? (tgt - head) - tv * kN : 0;
  for (; first < end; first += kGradThreads * kGradBatch) {
#pragma unroll
    for (int u = 0; u < kGradBatch; ++u) {
      const int i = first + u * kGradThreads;
      if (i >= end) break;
      float v[kN];
      unpack16<T>(w[u], v);
      const int nx = i + kGradThreads * kGradBatch;
      if (nx < end) load_one(nx, w[u]);
#pragma unroll
      for (int e = 0; e < kN; ++e) v[e] = one(v[e]);
      if (i == tv) {
#pragma unroll
        for (int e = 0; e < kN; ++e)
          if (e == te) v[e] = dl + v[e];
      }
      store16(g + head + (long)i * kN, v);
    }
  }
}

// -------------------------------------------------------------- launches --

template <typename T, int THREADS>
cudaError_t launch_logprobs(const LogprobArgs& a, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.rows * a.slices));
  cfg.blockDim = dim3(THREADS);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  if (a.slices > 1) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)a.slices;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
  }
  return cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, THREADS>, a);
}

template <typename T>
cudaError_t run_logprobs(const LogprobArgs& a, cudaStream_t st) {
  // a row that gives 512 threads less than two vectors each goes to 128; few rows
  // to 512 (one row of 32000 fp32: 5.9 us, with 256 threads 7.0), many to 256, several
  // rows an SM at a time (8192 rows: 167 us, with 512 threads 227)
  if (a.vocab / Vec<T>::kN < 1024) return launch_logprobs<T, 128>(a, st);
  return a.rows < 2 * 148 ? launch_logprobs<T, 512>(a, st) : launch_logprobs<T, 256>(a, st);
}

template <typename T>
cudaError_t run_grad(LogprobGradArgs a, cudaStream_t st) {
  const int per_cta = kGradThreads * kGradBatch * kGradLoops * Vec<T>::kN;
  a.per_row = (a.vocab + per_cta - 1) / per_cta;
  token_logprobs_grad_kernel<T><<<(unsigned)((long)a.rows * a.per_row), kGradThreads, 0, st>>>(a);
  return cudaGetLastError();
}

int bad(mxq_context* c, const char* msg) { return ctx_fail(c, MXQ_ERR_INVALID_ARGUMENT, msg); }

bool bad_shape(size_t rows, size_t vocab) {
  return vocab == 0 || vocab > (1u << 24) || rows > (1u << 24);
}

}  // namespace
}  // namespace mxq

using namespace mxq;

extern "C" {

int mxq_token_logprobs(mxq_ctx c, int dtype, const void* logits, size_t row_stride, size_t rows, size_t vocab,
                       const int32_t* target, size_t top_k, float* logp, float* entropy, float* lse, float* top_logp,
                       int32_t* top_ids) {
  if (!c) return bad(nullptr, "null context");
  const size_t es = dtype_bytes(dtype);
  if (!es) return bad(c, "token logprobs: unknown row type");
  if (bad_shape(rows, vocab)) return bad(c, "token logprobs: bad shape");
  if (top_k > MXQ_TOPK_MAX || top_k > vocab) return bad(c, "token logprobs: top_k exceeds 32 or the vocabulary");
  if (rows == 0) return MXQ_OK;
  if (!logits || !target || (top_k && (!top_logp || !top_ids))) return bad(c, "token logprobs: null pointer");
  if (row_stride < vocab) return bad(c, "token logprobs: rows overlap");
  if (reinterpret_cast<uintptr_t>(logits) % es) return bad(c, "token logprobs: misaligned logits");
  ServeDevice g(ctx_device(c));
  LogprobArgs a{logits, (long)row_stride, (int)rows, (int)vocab, (int)top_k, 1,
                target, logp, entropy, lse, top_logp, top_ids};
  // a long row is cut into slices while the rows alone leave SMs idle: a cluster
  // costs 2 us more than one CTA, which reads 256 KB in that time
  while (a.slices < kMaxSlices && rows * (size_t)a.slices < 148 && vocab * es / (size_t)a.slices > (256u << 10)) a.slices *= 2;
  const cudaStream_t st = ctx_stream(c);
  const cudaError_t e = dtype == MXQ_DT_F32    ? run_logprobs<float>(a, st)
                        : dtype == MXQ_DT_BF16 ? run_logprobs<__nv_bfloat16>(a, st)
                                               : run_logprobs<__half>(a, st);
  return serve_launched(c, e, "token logprobs");
}

int mxq_token_logprobs_grad(mxq_ctx c, int dtype, const void* logits, size_t row_stride, size_t rows, size_t vocab,
                            const int32_t* target, const float* lse, const float* entropy, const float* dlogp,
                            const float* dentropy, void* dlogits, size_t grad_stride) {
  if (!c) return bad(nullptr, "null context");
  const size_t es = dtype_bytes(dtype);
  if (!es) return bad(c, "token logprobs grad: unknown row type");
  if (bad_shape(rows, vocab)) return bad(c, "token logprobs grad: bad shape");
  if (rows == 0) return MXQ_OK;
  if (!logits || !target || !lse || !dlogits || (dentropy && !entropy))
    return bad(c, "token logprobs grad: null pointer");
  if (row_stride < vocab || grad_stride < vocab) return bad(c, "token logprobs grad: rows overlap");
  if (reinterpret_cast<uintptr_t>(logits) % es || reinterpret_cast<uintptr_t>(dlogits) % es)
    return bad(c, "token logprobs grad: misaligned rows");
  ServeDevice g(ctx_device(c));
  LogprobGradArgs a{logits, dlogits, (long)row_stride, (long)grad_stride, (int)rows, (int)vocab, 1,
                    target, lse, entropy, dlogp, dentropy};
  const cudaStream_t st = ctx_stream(c);
  const cudaError_t e = dtype == MXQ_DT_F32    ? run_grad<float>(a, st)
                        : dtype == MXQ_DT_BF16 ? run_grad<__nv_bfloat16>(a, st)
                                               : run_grad<__half>(a, st);
  return serve_launched(c, e, "token logprobs grad");
}

}  // extern "C"
