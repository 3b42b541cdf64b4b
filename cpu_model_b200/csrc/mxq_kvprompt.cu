// mxq_kvprompt.cu -- attention of prompts' rows (bf16 or fp16) over the paged
// 8-bit K/V cache, on tcgen05 with S, P and O in tensor memory.
//
// A unit is 256 query rows of one request and K/V head (tokens x the head's
// query heads), two M = 128 tiles A and B that share every K/V tile of 128 keys
// and take it in two steps of 64.
// int8 values are exact in fp16, and so is a bf16 row of q once a power of two
// has brought its largest element to 2^15 (what fp16 then rounds is below 2^-39 of it),
// so S = q K^T has fp32's accuracy.  The scales are applied where they cost
// nothing: K's and the row's in the fused multiply-add before exp (a block is 32 columns of
// S, its scale a constant of them), V's exactly in the conversion.  O += P V
// runs in fp16 too: P keeps 11 bits, and V' = q_v 2^(e_v - e + 8), e the unit's
// largest V exponent, is exact while the unit's exponents lie within 2^32 of
// each other.  Where they do not, that unit's P and V are bf16, which takes any
// exponent, and P is the sum of two terms of 8 bits, each with a product of its own.
//
// Warps: 0-3 and 4-7 softmax of tile A and of B, a row a thread; 8-11 bring K
// and V from their pages, int8 -> 16 bits, into two-stage rings in the 128-byte
// swizzle; 12 issues the MMAs of A and 13 those of B (an MMA takes a warp about
// 100 cycles to issue, more than the tensor cores need for it); 14 and 15 only fill the
// warpgroup, which gives its registers to the softmax.  P takes the columns of S that it was made
// from and is the MMA's A operand in tensor memory.  S of a step has one of two
// places, so the next step's is there when the softmax gets to it.  The rows of K are stored in the order of
// V's 16-byte pieces (token 8 j + 2 c + b of a block is key 8 c + 2 j + b), so
// neither is shuffled.  A row's maximum is only raised when it grows by 2^8:
// P stays below 2^15, O is rescaled rarely, and the end result is the same.
//
// Units are handed out one by one, the longest of each request first.  Every
// wait is bounded; one that gives up sets the status word and lets all roles
// run to the end without waiting.
//
// 4 prompts of 1142 to 1570 rows after 599 to 2839 tokens, 32 heads over 8 of 128,
// bf16: 285 us, 695 TFLOP/s, 42 % of cuBLAS's bf16 rate.  Latency bounds it: a
// softmax step's chain (S, maximum, exp, P, hand-over; without the exp 20 us less), and
// 15 us of each unit's start and end, about 4.6 units a CTA.  Units are not cut along
// the keys: 512 rows behind 32k tokens, 64 units, take 664 us, 4 times their operations'.
#include "mxq_serve.cuh"

namespace mxq {

namespace {

constexpr int kPromptThreads = 16 * 32;
constexpr int kTileKeys = 128;                    // keys the converters bring at a time
constexpr int kStepKeys = 64;                     // keys of an S
constexpr uint32_t kColS = 0, kColO = 256;        // TMEM columns: S of A, S of B, O of A, O of B
constexpr float kRise = 8.0f;                     // log2 of what P may grow by before O is rescaled
constexpr float kLift = 7.0f;                     // P starts at 2^7: fp16 has it normal down to 2^-21 of the maximum

#define MXQ_R4(a, i) "=r"(a[i]), "=r"(a[i + 1]), "=r"(a[i + 2]), "=r"(a[i + 3])
#define MXQ_W4(a, i) "r"(a[i]), "r"(a[i + 1]), "r"(a[i + 2]), "r"(a[i + 3])
__device__ __forceinline__ void tmem_ld32(uint32_t at, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,"
      "%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : MXQ_R4(r, 0), MXQ_R4(r, 4), MXQ_R4(r, 8), MXQ_R4(r, 12), MXQ_R4(r, 16), MXQ_R4(r, 20), MXQ_R4(r, 24), MXQ_R4(r, 28)
      : "r"(at));
}
__device__ __forceinline__ void tmem_st32(uint32_t at, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::MXQ_W4(r, 0), MXQ_W4(r, 4), MXQ_W4(r, 8), MXQ_W4(r, 12),
      MXQ_W4(r, 16), MXQ_W4(r, 20), MXQ_W4(r, 24), MXQ_W4(r, 28), "r"(at)
      : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t at, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : MXQ_R4(r, 0), MXQ_R4(r, 4), MXQ_R4(r, 8), MXQ_R4(r, 12)
      : "r"(at));
}
__device__ __forceinline__ void tmem_st16(uint32_t at, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::MXQ_W4(r, 0),
      MXQ_W4(r, 4), MXQ_W4(r, 8), MXQ_W4(r, 12), "r"(at)
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// D[tmem] (+)= A[tmem] * B[smem]^T, 16-bit inputs, fp32 accumulate.
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Instruction descriptor: bf16 or fp16 inputs, fp32 accumulator, both K-major.
__host__ __device__ constexpr uint32_t idesc_16(bool bf16, int M, int N) {
  return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

// Four int8 as two pairs of 16-bit numbers, exact.
__device__ __forceinline__ void widen_bf16(uint32_t w, uint32_t& a, uint32_t& b) {
  // 128 + the low seven bits, less 128 or (sign bit set) 256
  const uint32_t x = __byte_perm(w, 0u, 0x4140), y = __byte_perm(w, 0u, 0x4342);
  const uint32_t xp = (x & 0x007F007Fu) | 0x43004300u, xm = (x & 0x00800080u) | 0xC300C300u;
  const uint32_t yp = (y & 0x007F007Fu) | 0x43004300u, ym = (y & 0x00800080u) | 0xC300C300u;
  asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(a) : "r"(xp), "r"(xm));
  asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(b) : "r"(yp), "r"(ym));
}
__device__ __forceinline__ void widen_f16(uint32_t w, uint32_t& a, uint32_t& b) {
  // 1024 + (x + 128), less 1152
  w ^= 0x80808080u;
  const uint32_t x = __byte_perm(w, 0x64646464u, 0x4140), y = __byte_perm(w, 0x64646464u, 0x4342);
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(a) : "r"(x), "r"(0xE480E480u));
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(b) : "r"(y), "r"(0xE480E480u));
}
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t s) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(s));
  return r;
}

__device__ __forceinline__ int uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }

// Where a token of a block is among the K tile's rows (and so S's columns).
__host__ __device__ __forceinline__ int key_row(int t) { return ((t >> 1) & 3) * 8 + (t >> 3) * 2 + (t & 1); }
__host__ __device__ __forceinline__ int key_token(int row) { return ((row & 7) >> 1) * 8 + (row >> 3) * 2 + (row & 1); }

// Pairs of fp32 in one instruction, and the largest of three.
__device__ __forceinline__ uint64_t pair(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& x, float& y) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t s) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(s));
  return r;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// What rounding to bf16 took off a pair.
__device__ __forceinline__ uint32_t rest_bf16(uint32_t rounded, float lo, float hi) {
  return pack_bf16(lo - __uint_as_float(rounded << 16), hi - __uint_as_float(rounded & 0xFFFF0000u));
}
// 2^e in fp16 (0 below its smallest), e <= 8.
__device__ __forceinline__ uint32_t f16_pow2(int e) {
  return e >= -14 ? (uint32_t)(e + 15) << 10 : e >= -24 ? 1u << (e + 24) : 0u;
}
// 2^e in bf16 (0 below its smallest).
__device__ __forceinline__ uint32_t bf16_pow2(int e) {
  return e >= -126 ? (uint32_t)(e + 127) << 7 : e >= -133 ? 1u << (e + 133) : 0u;
}

template <int D>
struct PromptShared {
  static constexpr int kQTile = 128 * D * 2;      // one M tile of q, D / 64 halves of 128 rows x 128 bytes
  static constexpr int kKTile = kTileKeys * D * 2;
  static constexpr int kBytes = 2 * kQTile + 4 * kKTile;
};

struct Bars {
  uint64_t kfull[2], kempty[2], vfull[2], vempty[2], qfull[2], drain;
  uint64_t sfull[2][2], pfull[2][2], pvdone[2][2];   // [A, B][place]: two steps may be under way
};

// What the softmax needs of a K/V tile's blocks; four tiles deep: the
// converters are at most two ahead of the softmax.
struct TileNotes {
  float f[4];                            // 2^e_k, NaN for a NaN block
  uint32_t flags;                        // bit i: block i holds keys; bit 4 + i: its V is NaN
};

template <int D, bool kBf16>
__global__ void __launch_bounds__(kPromptThreads, 1) kv_prompt_kernel(KvPromptArgs a) {
  using S = PromptShared<D>;
  constexpr int kU = D / 16;             // 16-byte pieces of K, and of V, a converter thread has of a tile
  extern __shared__ __align__(1024) uint8_t raw_sm[];
  uint8_t* sm = raw_sm + ((1024u - (smem_u32(raw_sm) & 1023u)) & 1023u);
  uint8_t* sq = sm;
  uint8_t* sk = sm + 2 * S::kQTile;
  uint8_t* sv = sk + 2 * S::kKTile;
  int* s_sum = reinterpret_cast<int*>(sm + S::kBytes);             // [R + 1] units before a request
  __shared__ Bars bar;
  __shared__ TileNotes notes[4];
  __shared__ uint32_t s_tmem;
  __shared__ int s_unit[2];
  __shared__ int s_scan[kPromptThreads / 32];
  __shared__ int s_top[4], s_low[4];     // largest and smallest V scale byte of the unit, by converter warp
  __shared__ volatile int s_dead;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int G = a.G, Hkv = a.c.heads, nb = a.c.nb;
  auto start_of = [&](int r) { return min(max(a.cu[r], 0), a.n); };

  if (warp == 12) tmem_alloc(&s_tmem, 512);
  if (tid == 0) {
    s_dead = 0;
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar.kfull[i], 4);
      mbar_init(&bar.kempty[i], 2);
      mbar_init(&bar.vfull[i], 4);
      mbar_init(&bar.vempty[i], 2);
      for (int b = 0; b < 2; ++b) {
        mbar_init(&bar.pvdone[i][b], 1);
        mbar_init(&bar.sfull[i][b], 1);
        mbar_init(&bar.pfull[i][b], 4);
      }
    }
    mbar_init(&bar.qfull[0], 4);
    mbar_init(&bar.qfull[1], 4);
    mbar_init(&bar.drain, 2);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  // ---- units of the requests that this kernel takes
  {
    int base = 0;
    for (int r0 = 0; r0 < a.R; r0 += kPromptThreads) {
      const int r = r0 + tid;
      int w = 0;
      if (r < a.R) {
        const int rows = (start_of(r + 1) - start_of(r)) * G;
        if (rows > a.few && a.ctx_len[r] > 0) w = (rows + 255) / 256 * Hkv;
      }
      int s = w;
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += u;
      }
      __syncthreads();
      if (lane == 31) s_scan[warp] = s;
      __syncthreads();
      int before = base;
      for (int i = 0; i < kPromptThreads / 32; ++i) {
        if (i < warp) before += s_scan[i];
        base += s_scan[i];
      }
      if (r < a.R) s_sum[r] = before + s - w;
    }
    if (tid == 0) s_sum[a.R] = base;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  const int units = s_sum[a.R];

  // A hand-over comes soon, as a rule: 32 polls that do not put the warp to sleep first
  // (4 prompts of 900 to 2048 rows: 291 us without, 282 with 8, 280 with 32, 284 with 64).
  // Lanes may leave at different polls: a wait that an instruction of the whole warp
  // (tcgen05.ld, .st and .wait, bar.sync) follows has a __syncwarp behind it.
  auto wait = [&](uint64_t* b, uint32_t parity) {
    for (int i = 0; i < 32; ++i)
      if (mbar_test_wait(b, parity & 1u)) return;
    if (!s_dead && !mbar_wait(b, parity & 1u, a.status)) s_dead = 1;
  };

  // largest and smallest V scale byte of the unit (NaN and all-zero blocks aside)
  auto v_range = [&]() {
    return make_int2(max(max(s_top[0], s_top[1]), max(s_top[2], s_top[3])),
                     min(min(s_low[0], s_low[1]), min(s_low[2], s_low[3])));
  };
  // ---- the next unit: what every role needs of it
  struct Unit {
    int req, row0, rows, ctx, head, first, past;
    int see_a, see_b, na, nb, n;         // keys that the last row of A and of B sees, their steps; K/V tiles
  };
  uint32_t round = 0;
  auto next = [&](Unit& u) {
    if (tid == 0) s_unit[round & 1] = (int)atomicAdd(a.next, 1u);
    __syncwarp();
    asm volatile("bar.sync 1, %0;" ::"n"(kPromptThreads) : "memory");   // the last unit is done with shared and tensor memory
    const int id = s_unit[round & 1];
    ++round;
    if (id >= units) return false;
    int x = 0, y = a.R;
    while (y - x > 1) {
      const int mid = (x + y) >> 1;
      if (s_sum[mid] <= id) x = mid;
      else y = mid;
    }
    u.req = x;
    u.row0 = start_of(x);
    u.rows = (start_of(x + 1) - u.row0) * G;
    u.ctx = a.ctx_len[x];
    const int in = id - s_sum[x], tiles = (u.rows + 255) / 256;
    u.head = in % Hkv;
    u.first = (tiles - 1 - in / Hkv) * 256;
    u.past = u.ctx - u.rows / G;
    const int end_a = min(u.first + 128, u.rows), end_b = min(u.first + 256, u.rows);
    u.see_a = table_keys(a.c, a.max_pages, min(u.ctx, u.past + (end_a - 1) / G + 1));
    u.see_b = end_b > u.first + 128 ? table_keys(a.c, a.max_pages, min(u.ctx, u.past + (end_b - 1) / G + 1)) : 0;
    u.na = ceil_div(u.see_a, kStepKeys);
    u.nb = ceil_div(u.see_b, kStepKeys);
    u.n = (max(u.na, u.nb) + 1) >> 1;
    return true;
  };
  // registers: 256 x 168 + 128 x 112 + 128 x 56 = 64512 of the launch's 512 x 128
  uint32_t kt = 0;                       // K/V tiles of this CTA so far
  Unit un;

  if (warp < 8) {
    // ---------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
    uint32_t taken0 = 0, taken1 = 0;     // S taken from each place, and so P left there
    for (; next(un); kt += un.n) {
      const int x = warp >> 2, my = x ? un.nb : un.na;
      const int row0 = un.row0, head = un.head, past = un.past;
      const int row = un.first + x * 128 + (tid & 127);
      const bool valid = row < un.rows;
      const int t = row / G, h = head * G + (row - t * G);
      // the row of q, 16 bytes at a time, into its swizzled place, as fp16
      float qs = fabsf(a.scale2);                // |scale| log2(e) over the row's power of two
      {
        uint8_t* to = sq + x * S::kQTile;
        const uint16_t* from = static_cast<const uint16_t*>(a.q) + (long)(row0 + t) * a.q_stride + (long)h * D;
        const uint32_t flip = a.scale2 < 0.0f ? 0x80008000u : 0u;
        uint4 w[D / 8];
#pragma unroll
        for (int ch = 0; ch < D / 8; ++ch) {
          w[ch] = make_uint4(0, 0, 0, 0);
          if (valid) w[ch] = __ldg(reinterpret_cast<const uint4*>(from) + ch);
        }
        uint32_t top = 0;                        // the largest |q|, as its type's bits
#pragma unroll
        for (int ch = 0; ch < D / 8; ++ch) {
          const uint32_t m0 = __vmaxu2(w[ch].x & 0x7FFF7FFFu, w[ch].y & 0x7FFF7FFFu);
          top = __vmaxu2(top, __vmaxu2(m0, __vmaxu2(w[ch].z & 0x7FFF7FFFu, w[ch].w & 0x7FFF7FFFu)));
        }
        top = max(top & 0xFFFFu, top >> 16);
        const bool finite = top < (kBf16 ? 0x7F80u : 0x7C00u);
        float lift = 1.0f;
        if (kBf16 && finite) {
          // 2^(14 - exponent): |q| below 2^15
          const int up = min(14 - ((int)(top >> 7) - 127), 126);
          lift = __int_as_float((up + 127) << 23);
          qs *= __int_as_float((127 - up) << 23);
        }
        if (!finite) qs = __int_as_float(0x7fc00000);      // a row with an inf or a NaN is NaN by its scale
#pragma unroll
        for (int ch = 0; ch < D / 8; ++ch) {
          uint32_t v[4] = {w[ch].x ^ flip, w[ch].y ^ flip, w[ch].z ^ flip, w[ch].w ^ flip};
          if (kBf16)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = pack_f16(__uint_as_float(v[e] << 16) * lift, __uint_as_float(v[e] & 0xFFFF0000u) * lift);
          if (!finite) v[0] = v[1] = v[2] = v[3] = 0;
          *reinterpret_cast<uint4*>(to + (ch >> 3) * (128 * 128) + sw128_offset(tid & 127, ch & 7)) = make_uint4(v[0], v[1], v[2], v[3]);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar.qfull[x]);
      }
      const uint32_t quad = (uint32_t)(warp & 3) << 21;               // lane 32 * (warp % 4) of tensor memory
      const uint32_t ts = tmem + quad + kColS + x * 128, to = tmem + quad + kColO + x * 128;
      const int last = valid ? past + t : -1;
      float m = neg_inf(), l = 0.0f, unscale = 1.0f;
      bool half = true;
#pragma unroll 1
      for (int j = 0; j < my; ++j) {
        const int place = j & 1;
        const uint32_t tp = ts + place * 64;
        const uint32_t before = place ? taken0 : taken1;               // P left in the other place
        wait(&bar.sfull[x][place], place ? taken1 : taken0);
        __syncwarp();
        taken0 += place ^ 1;
        taken1 += place;
        tc_fence_after();
        uint32_t s0[32], s1[32];
        tmem_ld32(tp, s0);
        tmem_ld32(tp + 32, s1);
        const TileNotes& nt = notes[(kt + (j >> 1)) & 3];
        const uint32_t flags = nt.flags >> (2 * place);                // bits 0, 1: keys; 4, 5: NaN in V
        const float f0 = nt.f[2 * place] * qs, f1 = nt.f[2 * place + 1] * qs;
        const int limit = last - j * kStepKeys;  // keys 0 .. limit of the step are seen
        const bool cut = __any_sync(0xffffffffu, limit < kStepKeys - 1) || (flags & 3u) != 3u;
        // tokens of its two blocks that are seen: below these
        const int below0 = flags & 1u ? limit + 1 : 0, below1 = flags & 2u ? limit - 31 : 0;
        tmem_ld_wait();
        float u[4] = {neg_inf(), neg_inf(), neg_inf(), neg_inf()};
        if (!cut) {
#pragma unroll
          for (int c = 0; c < 32; c += 4) {
            u[0] = max3(u[0], __uint_as_float(s0[c]), __uint_as_float(s0[c + 1]));
            u[1] = max3(u[1], __uint_as_float(s0[c + 2]), __uint_as_float(s0[c + 3]));
            u[2] = max3(u[2], __uint_as_float(s1[c]), __uint_as_float(s1[c + 1]));
            u[3] = max3(u[3], __uint_as_float(s1[c + 2]), __uint_as_float(s1[c + 3]));
          }
        } else {
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            if (key_token(c) < below0) u[0] = fmaxf(u[0], __uint_as_float(s0[c]));
            if (key_token(c) < below1) u[2] = fmaxf(u[2], __uint_as_float(s1[c]));
          }
        }
        u[0] = fmaxf(u[0], u[1]);
        u[2] = fmaxf(u[2], u[3]);
        // nothing seen is no 0 (a scale of 0 times -inf)
        const float top = fmaxf(u[0] > neg_inf() ? u[0] * f0 : u[0], u[2] > neg_inf() ? u[2] * f1 : u[2]);
        const bool raise = top > (m == neg_inf() ? m : m + kRise);
        if (__any_sync(0xffffffffu, raise)) {
          const float mn = raise ? top : m;
          const float alpha = m == neg_inf() || !raise ? 1.0f : ex2(m - mn);   // a row without keys so far has O = 0
          l *= alpha;
          m = mn;
          if (j > 0) {
            // the product before this one; the one before that ended before this S began
            wait(&bar.pvdone[x][place ^ 1], before - 1);
            __syncwarp();
            tc_fence_after();
#pragma unroll 1
            for (int k = 0; k < D / 16; ++k) {
              uint32_t r[16];
              tmem_ld16(to + k * 16, r);
              tmem_ld_wait();
#pragma unroll
              for (int c = 0; c < 16; ++c) r[c] = __float_as_uint(__uint_as_float(r[c]) * alpha);
              tmem_st16(to + k * 16, r);
            }
            tmem_st_wait();
          }
        }
        const float base = m == neg_inf() ? 0.0f : m - kLift;
        if (j == 0) {
          wait(&bar.vfull[kt & 1], kt >> 1);     // the unit's V exponents are known
          __syncwarp();
          const int2 e = v_range();
          half = e.x - e.y <= 32;
          unscale = pow2_exact(e.x - 127 - 8);
        }
        uint32_t p[32];
        if (!cut && half && !(flags & 0x30u)) {  // the common step
          const uint64_t nb2 = pair(-base, -base), f02 = pair(f0, f0), f12 = pair(f1, f1);
          uint64_t part0 = 0, part1 = 0;
#pragma unroll
          for (int c = 0; c < 32; c += 2) {
            float p0, p1, q0, q1;
            unpair(fma2(pair(__uint_as_float(s0[c]), __uint_as_float(s0[c + 1])), f02, nb2), p0, p1);
            unpair(fma2(pair(__uint_as_float(s1[c]), __uint_as_float(s1[c + 1])), f12, nb2), q0, q1);
            p0 = ex2(p0);
            p1 = ex2(p1);
            q0 = ex2(q0);
            q1 = ex2(q1);
            part0 = add2(part0, pair(p0, p1));
            part1 = add2(part1, pair(q0, q1));
            p[c / 2] = pack_f16(p0, p1);
            p[16 + c / 2] = pack_f16(q0, q1);
          }
          float p0, p1;
          unpair(add2(part0, part1), p0, p1);
          l += p0 + p1;
        } else {
          float part0 = 0.0f, part1 = 0.0f;
          auto four = [&](int c, float (&y)[4]) {  // columns c, c + 1 of both blocks
            y[0] = ex2(fmaf(__uint_as_float(s0[c]), f0, -base)), y[1] = ex2(fmaf(__uint_as_float(s0[c + 1]), f0, -base));
            y[2] = ex2(fmaf(__uint_as_float(s1[c]), f1, -base)), y[3] = ex2(fmaf(__uint_as_float(s1[c + 1]), f1, -base));
            if (key_token(c) >= below0) y[0] = 0.0f;
            if (key_token(c + 1) >= below0) y[1] = 0.0f;
            if (key_token(c) >= below1) y[2] = 0.0f;
            if (key_token(c + 1) >= below1) y[3] = 0.0f;
            part0 += y[0] + y[1];
            part1 += y[2] + y[3];
          };
          if (half) {
#pragma unroll
            for (int c = 0; c < 32; c += 2) {
              float y[4];
              four(c, y);
              p[c / 2] = pack_f16(y[0], y[1]);
              p[16 + c / 2] = pack_f16(y[2], y[3]);
            }
          } else {
            uint32_t rest[32];                   // what bf16 rounds off P
#pragma unroll
            for (int c = 0; c < 32; c += 2) {
              float y[4];
              four(c, y);
              p[c / 2] = pack_bf16(y[0], y[1]);
              p[16 + c / 2] = pack_bf16(y[2], y[3]);
              rest[c / 2] = rest_bf16(p[c / 2], y[0], y[1]);
              rest[16 + c / 2] = rest_bf16(p[16 + c / 2], y[2], y[3]);
            }
            tmem_st32(tp + 32, rest);            // beside P: the step's S had 64 columns, P has 32
          }
          // a NaN block of V makes NaN of every row that sees a key of it
          if (((flags & 0x10u) && below0 > 0) || ((flags & 0x20u) && below1 > 0)) unscale = __int_as_float(0x7fc00000);
          l += part0 + part1;
        }
        tmem_st32(tp, p);                        // over S, which has been read
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar.pfull[x][place]);
      }
      if (my > 0) {
        const bool second = !(my & 1);
        wait(&bar.pvdone[x][second], (second ? taken1 : taken0) - 1);   // the last product, and so all
        __syncwarp();
        tc_fence_after();
      }
      const float inv = l == 0.0f ? 0.0f : unscale / l;
      const long at = (long)(row0 + t) * a.Hq + h;
#pragma unroll 1
      for (int k = 0; k < D / 32; ++k) {
        uint32_t r[32];
        if (my > 0) {
          tmem_ld32(to + k * 32, r);
          tmem_ld_wait();
        }
        if (valid) {
          uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + at * D + k * 32);
#pragma unroll
          for (int c = 0; c < 32; c += 8) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float y0 = my > 0 ? __uint_as_float(r[c + 2 * e]) * inv : 0.0f;
              const float y1 = my > 0 ? __uint_as_float(r[c + 2 * e + 1]) * inv : 0.0f;
              w[e] = kBf16 ? pack_bf16(y0, y1) : pack_f16(y0, y1);
            }
            dst[c / 8] = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
        __syncwarp();                            // rows that are not there are back for the next load
      }
      if (valid && a.lse) a.lse[at] = l == 0.0f ? neg_inf() : (m - kLift) * kLn2 + logf(l);
      tc_fence_before();                         // O may be written over after the next unit's barrier
    }
  } else if (warp < 12) {
    // ------------------------------------------------------- converters
    asm volatile("setmaxnreg.dec.sync.aligned.u32 112;");
    for (; next(un); kt += un.n) {
      const int w = warp - 8, ct = tid - 256, req = un.req, head = un.head, n = un.n;
      const int nblk = ceil_div(max(un.see_a, un.see_b), 32);
      // lanes 0-3: block 4 j + lane of tile j and its scales
      auto look = [&](int j, long& pl, uint32_t& sc) {
        pl = -1;
        sc = 0;
        const int b = 4 * j + lane, pg = b / nb;
        if (lane < 4 && b < nblk && pg < a.max_pages) {
          const int page = a.table[(long)req * a.max_pages + pg];
          if (page >= 0 && page < a.c.n_pages) {
            pl = kv_block(a.c, page, head, b - pg * nb);
            sc = (uint32_t)a.c.ks[pl] | (uint32_t)a.c.vs[pl] << 8;
          }
        }
      };
      uint4 kr[kU], vr[kU];
      // K: piece u of a thread is key u * kKeys + ct / (D / 16) of the tile, 16 dimensions of it
      constexpr int kKeys = 128 / (D / 16);      // keys a pass of the 128 threads: 16 or 32
      const int kq = ct / (D / 16), col = ct % (D / 16);
      auto load_k = [&](long pl) {
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const long at = __shfl_sync(0xffffffffu, pl, b);
          const uint4* from = reinterpret_cast<const uint4*>(a.c.k + at * (32 * D)) + kq * (D / 16) + col;
#pragma unroll
          for (int u = 0; u < 32 / kKeys; ++u) {
            uint4 w = make_uint4(0, 0, 0, 0);
            if (at >= 0) w = __ldg(from + u * 128);
            kr[b * (32 / kKeys) + u] = w;
          }
        }
      };
      // V: piece u is dimensions 2 pair, 2 pair + 1 of block kb, tokens of group vc
      const int vc = lane & 3, vkb = (lane >> 2) & 1, vpr = lane >> 3;
      auto load_v = [&](long pl) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const long at = __shfl_sync(0xffffffffu, pl, q * 2 + vkb);
          const uint4* from = reinterpret_cast<const uint4*>(a.c.v + at * (32 * D)) + (w * 4 + vpr) * 4 + vc;
#pragma unroll
          for (int u = 0; u < kU / 2; ++u) {
            uint4 x = make_uint4(0, 0, 0, 0);
            if (at >= 0) x = __ldg(from + u * 64);
            vr[u * 2 + q] = x;
          }
        }
      };
      // places in the tiles: a K key of token t is row key_row(t) of its block;
      // passes of 16 keys alternate between rows r and r + 4 of the swizzle
      const int krow = key_row(kq);
      const uint32_t kcol = (uint32_t)(col >> 2) * (128 * 128);
      // lanes 4-7 of a quarter warp are in the other half (D = 128): they store
      // their pieces in the other order, so that the eight hit all banks
      const uint32_t swap = D == 128 ? (lane >> 2) & 1 : 0;
      const uint32_t kat = kcol + sw128_offset(krow, (col & 3) * 2 + swap), kat2 = kcol + sw128_offset(krow, (col & 3) * 2 + 1 - swap);
      const uint32_t vat = sw128_offset(2 * (w * 4 + vpr), vkb * 4 + vc), vat2 = sw128_offset(2 * (w * 4 + vpr) + 1, vkb * 4 + vc);
      long pl, pl_next;
      uint32_t sc, sc_next;
      look(0, pl, sc);
      if (n > 0) {
        load_k(pl);
        load_v(pl);
      }
      look(1, pl_next, sc_next);
      {
        int top = 1, low = 254;
        for (int b = ct; b < nblk; b += 128) {
          const int pg = b / nb, page = pg < a.max_pages ? a.table[(long)req * a.max_pages + pg] : -1;
          if (page >= 0 && page < a.c.n_pages) {
            const int v = a.c.vs[kv_block(a.c, page, head, b - pg * nb)];
            if (v > 0 && v < 255) top = max(top, v), low = min(low, v);
          }
        }
        top = __reduce_max_sync(0xffffffffu, top);
        low = __reduce_min_sync(0xffffffffu, low);
        if (lane == 0) s_top[w] = top, s_low[w] = low;
        __syncwarp();
        asm volatile("bar.sync 2, 128;" ::: "memory");
      }
      const int2 range = v_range();
      const bool half = range.x - range.y <= 32;
      for (int j = 0; j < n; ++j) {
        const uint32_t g = kt + j;
        const int st = g & 1;
        if (w == 0 && lane < 4) {
          const uint32_t ks = sc & 0xFF;
          notes[g & 3].f[lane] = pl < 0 ? 0.0f : e8m0_to_float(ks);
        }
        const uint32_t there = __ballot_sync(0xffffffffu, lane < 4 && pl >= 0);
        const uint32_t vnan = __ballot_sync(0xffffffffu, lane < 4 && pl >= 0 && (sc >> 8) == 255u);
        if (w == 0 && lane == 0) notes[g & 3].flags = there | vnan << 4;
        if (g >= 2) wait(&bar.kempty[st], (g >> 1) - 1);
        uint8_t* kd = sk + st * S::kKTile;
#pragma unroll
        for (int u = 0; u < kU; ++u) {
          uint32_t o[8];
          widen_f16(kr[u].x, o[0], o[1]);
          widen_f16(kr[u].y, o[2], o[3]);
          widen_f16(kr[u].z, o[4], o[5]);
          widen_f16(kr[u].w, o[6], o[7]);
          const uint4 lo = make_uint4(o[0], o[1], o[2], o[3]), hi = make_uint4(o[4], o[5], o[6], o[7]);
          // 16 keys a pass: 4 rows on (which turns bit 2 of the swizzle), then the next block
          const uint32_t up = kKeys == 32 ? u * 32 * 128 : (u >> 1) * 32 * 128 + (u & 1) * 4 * 128;
          const uint32_t turn = kKeys == 32 ? 0 : (u & 1) * 64;
          *reinterpret_cast<uint4*>(kd + (kat ^ turn) + up) = swap ? hi : lo;
          *reinterpret_cast<uint4*>(kd + (kat2 ^ turn) + up) = swap ? lo : hi;
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar.kfull[st]);
        if (j + 1 < n) load_k(pl_next);
        if (g >= 2) wait(&bar.vempty[st], (g >> 1) - 1);
        uint8_t* vd = sv + st * S::kKTile;
        // the blocks' steps as pairs; a NaN block's values count as 0 (its rows become NaN at their end instead)
        uint32_t step[2];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int vs = (int)(__shfl_sync(0xffffffffu, sc, q * 2 + vkb) >> 8);
          step[q] = vs == 255 ? 0u : half ? f16_pow2(vs - range.x + 8) : bf16_pow2(vs - range.x + 8);
          step[q] |= step[q] << 16;
        }
        auto store_v = [&](int u, const uint32_t (&o)[8]) {
          const uint32_t up = (u & 1) * (D * 128) + (u >> 1) * 32 * 128;
          *reinterpret_cast<uint4*>(vd + vat + up) = make_uint4(o[0], o[1], o[2], o[3]);
          *reinterpret_cast<uint4*>(vd + vat2 + up) = make_uint4(o[4], o[5], o[6], o[7]);
        };
        if (half) {
#pragma unroll
          for (int u = 0; u < kU; ++u) {
            uint32_t o[8];
            widen_f16(vr[u].x, o[0], o[1]);
            widen_f16(vr[u].y, o[2], o[3]);
            widen_f16(vr[u].z, o[4], o[5]);
            widen_f16(vr[u].w, o[6], o[7]);
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = mul_f16x2(o[e], step[u & 1]);
            store_v(u, o);
          }
        } else {
#pragma unroll
          for (int u = 0; u < kU; ++u) {
            uint32_t o[8];
            widen_bf16(vr[u].x, o[0], o[1]);
            widen_bf16(vr[u].y, o[2], o[3]);
            widen_bf16(vr[u].z, o[4], o[5]);
            widen_bf16(vr[u].w, o[6], o[7]);
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = mul_bf16x2(o[e], step[u & 1]);
            store_v(u, o);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar.vfull[st]);
        if (j + 1 < n) load_v(pl_next);
        pl = pl_next;
        sc = sc_next;
        look(j + 2, pl_next, sc_next);
      }
    }
  } else {
    // ----------------------------------------------------------- issuer
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    const int x = warp - 12;             // the tile that this warp issues for
    uint32_t np0 = 0, np1 = 0;           // P taken from each place
    for (; next(un); kt += un.n) {
      if (x > 1) continue;
      const int my = uniform(x ? un.nb : un.na), n = uniform(un.n) * 2;   // steps of this tile; of the unit, in whole K/V tiles
      const uint32_t kt0 = uniform(kt), tm = uniform(tmem);
      constexpr uint32_t kIdS = idesc_16(false, 128, kStepKeys);
      constexpr uint32_t kIdWide = idesc_16(true, 128, D);
      uint32_t id_o = idesc_16(false, 128, D);
      const uint64_t dq = sw128_kmajor_desc(smem_u32(sq + x * S::kQTile)), dk = sw128_kmajor_desc(smem_u32(sk)),
                     dv = sw128_kmajor_desc(smem_u32(sv));
      const uint32_t to = tm + kColO + x * 128;
      auto alive = [&]() { return __all_sync(0xffffffffu, !s_dead) != 0; };   // the same in all lanes
      wait(&bar.qfull[x], round - 1);
      // step i: the product of step i - 2, and S of step i, whose place it frees
#pragma unroll 1
      for (int i = 0; i < n + 2; ++i) {
        const int j = i - 2, place = i & 1;
        const uint32_t g = kt0 + (j >> 1), gk = kt0 + (i >> 1);
        const uint32_t ts = tm + kColS + x * 128 + place * 64;
        if (j >= 0 && !place) {
          wait(&bar.vfull[g & 1], g >> 1);
          const int2 e = v_range();
          id_o = e.x - e.y > 32 ? kIdWide : idesc_16(false, 128, D);
        }
        if (j >= 0 && j < my) {
          wait(&bar.pfull[x][place], place ? np1 : np0);
          np0 += place ^ 1;
          np1 += place;
          tc_fence_after();
          if (alive() && elect_one()) {
            // O += P of the step and its half of the V tile
            const uint64_t db = dv + (((g & 1) * S::kKTile + place * (D * 128)) >> 4);
#pragma unroll
            for (int k = 0; k < kStepKeys / 16; ++k) mma_ts(to, ts + k * 8, db + k * 2, id_o, j > 0 || k > 0);
            if (id_o == kIdWide)         // P's second term
#pragma unroll 1
              for (int k = 0; k < kStepKeys / 16; ++k) mma_ts(to, ts + 32 + k * 8, db + k * 2, kIdWide, 1);
            mma_commit(&bar.pvdone[x][place]);
          }
          __syncwarp();
        }
        if (i < n && !place) {
          wait(&bar.kfull[gk & 1], gk >> 1);
          tc_fence_after();
        }
        if (i < my && alive() && elect_one()) {
          // S: D / 16 MMAs of 32 bytes a row, a 16 KB half every four; the step's
          // keys are rows place * 64 .. of the K tile
          const uint64_t db = dk + (((gk & 1) * S::kKTile + place * (kStepKeys * 128)) >> 4);
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t at = ((k >> 2) * (128 * 128) + (k & 3) * 32) >> 4;
            mma_bf16_ss(ts, dq + at, db + at, kIdS, k > 0);
          }
          mma_commit(&bar.sfull[x][place]);
        }
        __syncwarp();
        // the tiles that this warp is done with
        if (place && alive() && elect_one()) {
          if (j >= 0) mma_commit(&bar.vempty[g & 1]);
          if (i < n) mma_commit(&bar.kempty[gk & 1]);
        }
        __syncwarp();
      }
    }
  }
  // ---- every MMA has ended before tensor memory goes
  if (warp == 12 || warp == 13) {
    if (elect_one()) mma_commit(&bar.drain);
    (void)mbar_wait(&bar.drain, 0, a.status);
    __syncwarp();
  }
  __syncthreads();
  if (warp == 12) tmem_dealloc(tmem, 512);
  // the last CTA leaves the counters at zero
  if (tid == 0 && atomicAdd(a.next + 1, 1u) == gridDim.x - 1) {
    a.next[0] = 0;
    a.next[1] = 0;
  }
}

template <int D, bool kBf16>
cudaError_t launch(const KvPromptArgs& a, int ctas, cudaStream_t st) {
  static SmemAttr attr;
  constexpr size_t kTiles = 1024 + PromptShared<D>::kBytes;
  static_assert(kTiles + (MXQ_KV_MAX_REQUESTS + 1) * 4 + 1536 <= 227 << 10, "every number of requests fits");
  const size_t smem = kTiles + ((size_t)a.R + 1) * 4;
  const cudaError_t e = attr.ensure(kv_prompt_kernel<D, kBf16>, smem);
  if (e != cudaSuccess) return e;
  kv_prompt_kernel<D, kBf16><<<(unsigned)ctas, kPromptThreads, smem, st>>>(a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_kv_prompt(const KvPromptArgs& a, int ctas, cudaStream_t st) {
  if (a.c.dim == 64) return a.bf16 ? launch<64, true>(a, ctas, st) : launch<64, false>(a, ctas, st);
  return a.bf16 ? launch<128, true>(a, ctas, st) : launch<128, false>(a, ctas, st);
}

}  // namespace mxq
