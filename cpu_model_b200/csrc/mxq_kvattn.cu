// mxq_kvattn.cu -- causal attention of new rows over the paged 8-bit K/V
// cache (mxq_kv.cu), on the int8 MMA.
//
// What a block holds is int8 with one power of two for its 32 tokens of a
// head, so both products can run in integers, exactly, on the bytes as they
// are stored:
//   S = q K^T: a query row is written once as a fixed-point number of two or
//   three signed base-256 digits (planes), q = 2^e sum_i 256^i q_i; rows 0-7 of an
//   m16n8k32 MMA take the upper digit of eight query rows and rows 8-15 the
//   lower, so a lane holds both digits' sums of its row and joins them itself:
//   s = 2^(e + e_k) scale (256 hi + lo).
//   O = P V: the block's probabilities, relative to the block's own maximum b
//   of the row, become such digits too, and O += 2^(e_v) 2^(b - m) (256 hi +
//   lo) / 32512.  The sums of a block fit int32 (127^2 * 32 * 256).
// 16-bit rows take two digits (15 bits; the error of a probability is 2^-16 of the
// block's largest, a 128th of bf16's rounding of the result), fp32 rows three.
// Lengths, maxima, sums and O are fp32.
//
// Fragments: B's columns are tokens (S) and dimensions (O).  The order of the
// summed index is free as long as A and B agree, so K rows are read 16 bytes a
// lane as stored, V was stored in the order in which S leaves its
// probabilities (eight tokens a lane), and nothing is shuffled.
//
// Work: (request, head, tile of query rows) x blocks, in one line that is cut
// into equal pieces, one a CTA (two CTAs an SM), whatever the lengths are;
// every CTA finds its piece by summing the lengths itself.  A piece's blocks go
// to the CTA's warps in turn, each with its own ring of cp.async stages and its own
// running maximum; they are joined through shared memory.  A tile that
// several CTAs share is joined by the last of them from workspace, in the order of
// the pieces, so the result does not depend on who was last.
#include "mxq_serve.cuh"

namespace mxq {

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kStages = 3;
constexpr int kMaxRows = 16;             // query rows a tile
constexpr int kMinPiece = 8;             // blocks a CTA at least
constexpr float kLn2 = 0.693147180559945f;

struct AttnArgs {
  KvView c;
  const void* q;
  void* out;
  float* lse;
  const int32_t *table, *ctx_len, *cu;
  long q_stride;
  int dtype, R, n, Hq, G, max_pages;
  float scale2;                          // scale * log2(e)
  uint32_t* counters;                    // [CTAs], zero
  float* part;                           // [CTAs][2][kMaxRows][D + 2]
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float neg_inf() { return -__int_as_float(0x7f800000); }

__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Shared memory of a CTA: the lengths' sums, the query rows' digits, and the
// warps' rings, whose place the joining of the warps takes afterwards.
template <int D, int MT, int NP>
struct Layout {
  static constexpr int kRows = 8 * MT;
  static constexpr int kQ = NP * kRows * D;                       // digits [plane][row][D]
  static constexpr int kStage = 64 * D;                           // one block's K and V
  static constexpr int kRing = kWarps * kStages * kStage;
  static constexpr int kJoin = kWarps * kRows * (D + 2) * 4;
  static constexpr int kBody = kRing > kJoin ? kRing : kJoin;
  static size_t bytes(int R) { return (size_t)kBody + kQ + kRows * 8 + ((size_t)R + 1) * 8 + 64; }
};

// Start of request r's rows (r = R: their end), inside q whatever is given.
__device__ __forceinline__ int row_start(const AttnArgs& a, int r) { return min(max(a.cu[r], 0), a.n); }

template <int D, int MT, int NP>
__global__ void __launch_bounds__(kThreads, 2) kv_attn_kernel(AttnArgs a) {
  using L = Layout<D, MT, NP>;
  constexpr int kRows = L::kRows;
  constexpr int kJ = D / 64;             // 64-dimension halves
  constexpr int kU = D / 16;             // V words of 16 dimensions
  constexpr int kTiles = NP == 2 ? MT : (MT == 1 ? 2 : 3);   // MMA row tiles
  extern __shared__ __align__(16) uint8_t sm[];
  uint8_t* s_q = sm + L::kBody;
  float* s_scale = reinterpret_cast<float*>(s_q + L::kQ);         // [kRows] 2^e scale log2(e)
  int* s_last = reinterpret_cast<int*>(s_scale + kRows);          // [kRows] last key a row sees
  long* s_sum = reinterpret_cast<long*>(s_last + kRows);          // [R + 1]
  __shared__ long s_warp[kWarps];
  __shared__ int s_flag;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int c4 = lane & 3, r8 = lane >> 2;
  const int Hkv = a.c.heads, G = a.G, nb = a.c.nb;

  // ---- the line of work: tiles * blocks * heads of every request, summed
  {
    long base = 0;
    for (int r0 = 0; r0 < a.R; r0 += kThreads) {
      const int r = r0 + tid;
      long w = 0;
      if (r < a.R) {
        const int rows = (row_start(a, r + 1) - row_start(a, r)) * G, len = a.ctx_len[r];
        if (rows > 0 && len > 0) w = (long)((rows + kRows - 1) / kRows) * ((len + 31) >> 5) * Hkv;
      }
      long s = w;
      for (int o = 1; o < 32; o <<= 1) {
        const long u = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += u;
      }
      __syncthreads();
      if (lane == 31) s_warp[warp] = s;
      __syncthreads();
      long before = base;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) {
        if (i < warp) before += s_warp[i];
        base += s_warp[i];
      }
      if (r < a.R) s_sum[r] = before + s - w;
    }
    if (tid == 0) s_sum[a.R] = base;
    __syncthreads();
  }
  // rows that no key is for: 0 and -inf
  {
    const int used = row_start(a, a.R);
    const long per = (long)a.Hq * (D / 4);
    const float zero[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (long i = (long)blockIdx.x * kThreads + tid; i < (long)(a.n - used) * per; i += (long)gridDim.x * kThreads) {
      store4_dt(a.dtype, a.out, (long)used * a.Hq * D + i * 4, zero);
      if (a.lse && i % (D / 4) == 0) a.lse[(long)used * a.Hq + i / (D / 4)] = neg_inf();
    }
    for (int r = blockIdx.x; r < a.R; r += gridDim.x) {
      if (a.ctx_len[r] > 0) continue;
      const long r0 = row_start(a, r), rn = row_start(a, r + 1) - r0;
      for (long i = tid; i < rn * per; i += kThreads) {
        store4_dt(a.dtype, a.out, r0 * a.Hq * D + i * 4, zero);
        if (a.lse && i % (D / 4) == 0) a.lse[r0 * a.Hq + i / (D / 4)] = neg_inf();
      }
    }
  }
  const long total = s_sum[a.R];
  long len = (total + gridDim.x - 1) / gridDim.x;
  if (len < kMinPiece) len = kMinPiece;
  const long lo = blockIdx.x * len, hi = min(lo + len, total);

  uint8_t* ring = sm + warp * (kStages * L::kStage);
  const uint32_t ring_s = smem_u32(ring);

  int req = 0;
  if (lo < hi) {                         // the request that holds block lo: the last with sum <= lo and work
    int x = 0, y = a.R;
    while (y - x > 1) {
      const int mid = (x + y) >> 1;
      if (s_sum[mid] <= lo) x = mid;
      else y = mid;
    }
    req = x;
  }
  for (long pos = lo; pos < hi;) {
    while (s_sum[req + 1] <= pos) ++req;
    const int row0 = row_start(a, req), rows = (row_start(a, req + 1) - row0) * G, ctx = a.ctx_len[req];
    const int nblk = (ctx + 31) >> 5, tiles = (rows + kRows - 1) / kRows;
    const long in = pos - s_sum[req];
    const int unit = (int)(in / nblk), b0 = (int)(in - (long)unit * nblk);
    const int head = unit / tiles, tile = unit - head * tiles;
    const long unit0 = pos - b0;
    const int take = (int)min((long)(nblk - b0), hi - pos);
    pos += take;
    const int nrows = min(kRows, rows - tile * kRows);
    const int past = ctx - rows / G;
    // keys that the tile's last row sees
    const int seen = min(ctx, past + (tile * kRows + nrows - 1) / G + 1);
    const int blocks = (seen + 31) >> 5;           // <= 0: none
    const int b1 = min(b0 + take, blocks);
    const long c_first = unit0 / len, c_last = blocks > 0 ? (unit0 + blocks - 1) / len : c_first;
    if (b0 >= b1 && !(blocks <= 0 && b0 == 0)) continue;

    // ---- this warp's blocks b0 + warp, + kWarps, ...: their places, 32 at a time
    const int mine = b1 > b0 + warp ? (b1 - b0 - warp + kWarps - 1) / kWarps : 0;
    long place = -1;                     // lane l: block l of the current 32
    uint32_t place_sc = 0;               // its scales: K | V << 8
    auto look_up = [&](int first) {
      const int i = first + lane;
      place = -1;
      place_sc = 0;
      if (i < mine) {
        const int b = b0 + warp + i * kWarps, pg = b / nb;
        const int page = pg < a.max_pages ? a.table[(long)req * a.max_pages + pg] : -1;
        if (page >= 0 && page < a.c.n_pages) {
          place = kv_block(a.c, page, head, b - pg * nb);
          place_sc = (uint32_t)a.c.ks[place] | (uint32_t)a.c.vs[place] << 8;
        }
      }
    };
    auto fetch = [&](int i) {            // block i of this warp into its stage
      const long at = __shfl_sync(0xffffffffu, place, i & 31);
      if (at >= 0) {
        const uint32_t st = ring_s + (i % kStages) * L::kStage;
        const int8_t* k = a.c.k + at * (32 * D);
        const int8_t* v = a.c.v + at * (32 * D);
#pragma unroll
        for (int u = 0; u < 2 * D / 32; ++u) {
          const int ch = u * 32 + lane;
          // rows of 128 bytes: every other row's halves change places, so that a
          // quarter warp's two rows lie in different banks
          const int sw = D == 128 ? ch ^ ((ch >> 3 & 1) << 2) : ch;
          cp16(st + sw * 16, k + ch * 16);
          cp16(st + 32 * D + ch * 16, v + ch * 16);
        }
      }
      cp_commit();
    };
    look_up(0);
    uint32_t sc_now = place_sc;
    long pl_now = place;
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) {
      if (i < mine) fetch(i);
      else cp_commit();
    }

    // ---- the query rows' digits
    for (int r = warp; r < kRows; r += kWarps) {
      float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      uint32_t top = 0;
      const int gr = tile * kRows + r, t = gr / G, h = head * G + (gr - t * G);
      if (r < nrows && lane < D / 4) {
        load4_dt(a.dtype, a.q, (long)(row0 + t) * a.q_stride + (long)h * D + lane * 4, x);
#pragma unroll
        for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
      }
      top = __reduce_max_sync(0xffffffffu, top);
      const bool finite = top < 0x7f800000u;
      // |digits| <= 127 * 256^(NP-1); tiny rows keep a step that is a normal number
      const int e = max(e8m0_exponent<127>(__uint_as_float(top)) - 8 * (NP - 1), -126);
      const float inv = finite ? __int_as_float((127 - e) << 23) : 0.0f;
      uint32_t dig[NP];
#pragma unroll
      for (int p = 0; p < NP; ++p) dig[p] = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        int q = finite ? __float2int_rn(x[i] * inv) : 0;
#pragma unroll
        for (int p = NP - 1; p >= 0; --p) {        // plane 0 is the uppermost
          dig[p] |= (uint32_t)(q & 0xFF) << (8 * i);
          q = (q + 128) >> 8;
        }
      }
      if (lane < D / 4)
#pragma unroll
        for (int p = 0; p < NP; ++p) *reinterpret_cast<uint32_t*>(s_q + (p * kRows + r) * D + lane * 4) = dig[p];
      if (lane == 0) {
        s_scale[r] = finite ? __int_as_float((e + 127) << 23) * a.scale2 : __int_as_float(0x7fc00000);
        s_last[r] = r < nrows ? past + t : -1;
      }
    }
    __syncthreads();

    // ---- A fragments: 64 dimensions are two k-steps; lane (r8, c4) has 16
    // bytes of a row: words 0, 1 of step 0 and 2, 3 of step 1
    uint4 qa[MT][NP][kJ];
    float qs[MT];
    int last[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
      for (int p = 0; p < NP; ++p)
#pragma unroll
        for (int j = 0; j < kJ; ++j)
          qa[m][p][j] = *reinterpret_cast<const uint4*>(s_q + (p * kRows + m * 8 + r8) * D + j * 64 + c4 * 16);
      qs[m] = s_scale[m * 8 + r8];
      last[m] = s_last[m * 8 + r8];
    }
    float o[MT][kU][4];
    float mx[MT], sum[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      mx[m] = neg_inf();
      sum[m] = 0.0f;
#pragma unroll
      for (int u = 0; u < kU; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[m][u][e] = 0.0f;
    }

    for (int i = 0; i < mine; ++i) {
      const int nx = i + kStages - 1;
      // sc_now / pl_now: the 32 blocks that hold block i; place / place_sc:
      // those that hold block nx
      if ((i & 31) == 0 && i) {
        sc_now = place_sc;
        pl_now = place;
      }
      if ((nx & 31) == 0) look_up(nx);
      cp_wait<kStages - 2>();
      __syncwarp();
      const uint8_t* st = ring + (i % kStages) * L::kStage;
      const long at = __shfl_sync(0xffffffffu, pl_now, i & 31);
      const uint32_t sc = __shfl_sync(0xffffffffu, sc_now, i & 31);
      if (at >= 0) {
        const float ks = e8m0_to_float(sc & 0xFF), vs = e8m0_to_float(sc >> 8);
        const int key0 = (b0 + warp + i * kWarps) * 32 + 2 * c4;
        int acc[kTiles][4][4];
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
#pragma unroll
          for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[t][n][e] = 0;
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int j = 0; j < kJ; ++j) {
            const int row = 8 * n + r8;
            const int ch = D == 128 ? row * 8 + ((j * 4 + c4) ^ ((row & 1) << 2)) : row * 4 + c4;
            const uint4 b = *reinterpret_cast<const uint4*>(st + ch * 16);
#pragma unroll
            for (int m = 0; m < MT; ++m) {
              mma_s8(acc[m][n], qa[m][0][j].x, qa[m][1][j].x, qa[m][0][j].y, qa[m][1][j].y, b.x, b.y);
              mma_s8(acc[m][n], qa[m][0][j].z, qa[m][1][j].z, qa[m][0][j].w, qa[m][1][j].w, b.z, b.w);
            }
            if (NP == 3) {
              const uint4 l0 = qa[0][NP - 1][j];
              const uint4 l1 = MT == 2 ? qa[MT - 1][NP - 1][j] : make_uint4(0, 0, 0, 0);
              mma_s8(acc[kTiles - 1][n], l0.x, l1.x, l0.y, l1.y, b.x, b.y);
              mma_s8(acc[kTiles - 1][n], l0.z, l1.z, l0.w, l1.w, b.z, b.w);
            }
          }
        uint32_t pa[MT][NP][2];          // probabilities' digits, slots 0-3 and 4-7
        float fac[MT], alpha[MT];
        bool same = true;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          float x[8];
          float bm = neg_inf();
          const float f = qs[m] * ks;
#pragma unroll
          for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int hl = acc[m][n][e] * 256 + acc[m][n][2 + e];
              float s = (float)hl;
              if (NP == 3) s = fmaf(s, 256.0f, (float)acc[kTiles - 1][n][2 * m + e]);
              s = key0 + 8 * n + e <= last[m] ? s * f : neg_inf();
              x[2 * n + e] = s;
              bm = fmaxf(bm, s);
            }
          bm = fmaxf(bm, __shfl_xor_sync(0xffffffffu, bm, 1));
          bm = fmaxf(bm, __shfl_xor_sync(0xffffffffu, bm, 2));
          const bool none = bm == neg_inf();
          const float mn = fmaxf(mx[m], bm), ms = mn == neg_inf() ? 0.0f : mn;
          const float beta = none ? 0.0f : ex2(bm - ms);
          alpha[m] = ex2(mx[m] - ms);
          same = same && mn == mx[m];
          const float bs = none ? 0.0f : bm;
          float ps = 0.0f;
          constexpr float kTop = NP == 2 ? 32512.0f : 8323072.0f;       // 127 * 256^(NP-1)
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float p = ex2(x[4 * g + e] - bs);
              ps += p;
              // the sum with 2^23 leaves the nearest integer in the low bits
              w[e] = __float_as_uint(fmaf(p, kTop, 8388608.0f));
            }
            if (NP == 3) w[0] &= 0x7fffffu, w[1] &= 0x7fffffu, w[2] &= 0x7fffffu, w[3] &= 0x7fffffu;
#pragma unroll
            for (int p = NP - 1; p >= 0; --p) {
              pa[m][p][g] = __byte_perm(__byte_perm(w[0], w[1], 0x0040), __byte_perm(w[2], w[3], 0x0040), 0x5410);
              if (p) {
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = (w[e] + 128) >> 8;
              }
            }
          }
          sum[m] = sum[m] * alpha[m] + ps * beta;
          mx[m] = mn;
          fac[m] = none ? 0.0f : beta * vs * (1.0f / kTop);
        }
        same = __all_sync(0xffffffffu, same);
        if (!same) {
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int u = 0; u < kU; ++u)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[m][u][e] *= alpha[m];
        }
        const uint8_t* sv = st + 32 * D;
#pragma unroll
        for (int u = 0; u < kU; ++u) {
          const uint4 b = *reinterpret_cast<const uint4*>(sv + ((8 * u + r8) * 4 + c4) * 16);
#pragma unroll
          for (int d = 0; d < 2; ++d) {
            const uint32_t b_lo = d ? b.z : b.x, b_hi = d ? b.w : b.y;
            int pv[kTiles][4];
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
#pragma unroll
              for (int e = 0; e < 4; ++e) pv[t][e] = 0;
#pragma unroll
            for (int m = 0; m < MT; ++m)
              mma_s8(pv[m], pa[m][0][0], pa[m][1][0], pa[m][0][1], pa[m][1][1], b_lo, b_hi);
            if (NP == 3)
              mma_s8(pv[kTiles - 1], pa[0][NP - 1][0], MT == 2 ? pa[MT - 1][NP - 1][0] : 0u, pa[0][NP - 1][1],
                     MT == 2 ? pa[MT - 1][NP - 1][1] : 0u, b_lo, b_hi);
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                float s = (float)(pv[m][e] * 256 + pv[m][2 + e]);
                if (NP == 3) s = fmaf(s, 256.0f, (float)pv[kTiles - 1][2 * m + e]);
                o[m][u][2 * e + d] = fmaf(s, fac[m], o[m][u][2 * e + d]);
              }
          }
        }
      }
      __syncwarp();                      // every lane has read stage i before it is refilled
      if (nx < mine) fetch(nx);
      else cp_commit();
    }
    cp_wait<0>();
    __syncthreads();                     // the rings are idle: their place takes the join

    // ---- the warps' results side by side: [warp][row][D], maxima and sums
    float* j_o = reinterpret_cast<float*>(sm);
    float* j_m = j_o + kWarps * kRows * D;
    float* j_l = j_m + kWarps * kRows;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int row = m * 8 + r8;
      float s = sum[m];
      s += __shfl_xor_sync(0xffffffffu, s, 1);
      s += __shfl_xor_sync(0xffffffffu, s, 2);
      if (row < nrows) {
        // lane (r8, c4) has dimensions 16 u + 4 c4 .. + 3
#pragma unroll
        for (int u = 0; u < kU; ++u)
          *reinterpret_cast<float4*>(j_o + (warp * kRows + row) * D + u * 16 + c4 * 4) =
              make_float4(o[m][u][0], o[m][u][1], o[m][u][2], o[m][u][3]);
        if (c4 == 0) {
          j_m[warp * kRows + row] = mx[m];
          j_l[warp * kRows + row] = s;
        }
      }
    }
    __syncthreads();

    const bool whole = c_first == c_last;
    // a piece that starts its tile and does not end it goes to slot 1 of the
    // CTA, one that continues a tile to slot 0: there is at most one of each
    const long slot_size = (long)kMaxRows * (D + 2);
    float* part = a.part + ((long)blockIdx.x * 2 + (blockIdx.x == c_first ? 1 : 0)) * slot_size;
    for (int w = tid; w < nrows * (D / 4); w += kThreads) {
      const int row = w / (D / 4), d = (w - row * (D / 4)) * 4;
      float m = neg_inf();
#pragma unroll
      for (int i = 0; i < kWarps; ++i) m = fmaxf(m, j_m[i * kRows + row]);
      const float ms = m == neg_inf() ? 0.0f : m;
      float l = 0.0f;
      float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < kWarps; ++i) {
        const float f = ex2(j_m[i * kRows + row] - ms);
        l += f * j_l[i * kRows + row];
        const float4 v = *reinterpret_cast<const float4*>(j_o + (i * kRows + row) * D + d);
        y[0] += f * v.x; y[1] += f * v.y; y[2] += f * v.z; y[3] += f * v.w;
      }
      if (whole) {
        const int gr = tile * kRows + row, t = gr / G, h = head * G + (gr - t * G);
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] *= inv;
        store4_dt(a.dtype, a.out, ((long)(row0 + t) * a.Hq + h) * D + d, y);
        if (a.lse && d == 0) a.lse[(long)(row0 + t) * a.Hq + h] = l == 0.0f ? neg_inf() : m * kLn2 + logf(l);
      } else {
        *reinterpret_cast<float4*>(part + row * D + d) = make_float4(y[0], y[1], y[2], y[3]);
        if (d == 0) {
          part[kMaxRows * D + row] = m;
          part[kMaxRows * (D + 1) + row] = l;
        }
      }
    }
    if (!whole) {
      __threadfence();
      __syncthreads();
      const int parts = (int)(c_last - c_first) + 1;
      if (tid == 0) {
        s_flag = atomicAdd(a.counters + c_first, 1u) == (uint32_t)parts - 1;
        if (s_flag) a.counters[c_first] = 0;
      }
      __syncthreads();
      if (s_flag) {
        __threadfence();
        for (int w = tid; w < nrows * (D / 4); w += kThreads) {
          const int row = w / (D / 4), d = (w - row * (D / 4)) * 4;
          float m = neg_inf(), l = 0.0f;
          float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
          for (int i = 0; i < parts; ++i) {
            const float* p = a.part + ((c_first + i) * 2 + (i == 0 ? 1 : 0)) * slot_size;
            const float pm = __ldcg(p + kMaxRows * D + row), pl = __ldcg(p + kMaxRows * (D + 1) + row);
            const float4 v = __ldcg(reinterpret_cast<const float4*>(p + row * D + d));
            const float mn = fmaxf(m, pm), ms = mn == neg_inf() ? 0.0f : mn;
            const float fa = ex2(m - ms), fb = ex2(pm - ms);
            l = l * fa + pl * fb;
            y[0] = y[0] * fa + v.x * fb; y[1] = y[1] * fa + v.y * fb;
            y[2] = y[2] * fa + v.z * fb; y[3] = y[3] * fa + v.w * fb;
            m = mn;
          }
          const int gr = tile * kRows + row, t = gr / G, h = head * G + (gr - t * G);
          const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] *= inv;
          store4_dt(a.dtype, a.out, ((long)(row0 + t) * a.Hq + h) * D + d, y);
          if (a.lse && d == 0) a.lse[(long)(row0 + t) * a.Hq + h] = l == 0.0f ? neg_inf() : m * kLn2 + logf(l);
        }
      }
    }
    __syncthreads();                     // the join's place goes back to the rings
  }
}

SmemAttr g_attn_attr[2][2][2];

template <int D, int MT, int NP>
cudaError_t launch(const AttnArgs& a, int ctas, cudaStream_t st) {
  const size_t smem = Layout<D, MT, NP>::bytes(a.R);
  const cudaError_t e = g_attn_attr[D == 128][MT - 1][NP - 2].ensure(kv_attn_kernel<D, MT, NP>, smem);
  if (e != cudaSuccess) return e;
  kv_attn_kernel<D, MT, NP><<<(unsigned)ctas, kThreads, smem, st>>>(a);
  return cudaGetLastError();
}

template <int D>
cudaError_t launch_d(const AttnArgs& a, bool two, bool f32, int ctas, cudaStream_t st) {
  if (two) return f32 ? launch<D, 2, 3>(a, ctas, st) : launch<D, 2, 2>(a, ctas, st);
  return f32 ? launch<D, 1, 3>(a, ctas, st) : launch<D, 1, 2>(a, ctas, st);
}

int bad(mxq_context* c, const char* msg) { return ctx_fail(c, MXQ_ERR_INVALID_ARGUMENT, msg); }

}  // namespace
}  // namespace mxq

using namespace mxq;

extern "C" {

int mxq_kv_attention(mxq_ctx c, const mxq_kv_cache* cache, int dtype, const void* q, size_t q_stride, size_t n,
                     size_t n_heads, const int32_t* table, size_t max_pages, const int32_t* ctx_len, const int32_t* cu,
                     size_t n_req, size_t max_new, float scale, void* out, float* lse) {
  if (!c) return bad(nullptr, "null context");
  KvView kv;
  if (const char* msg = kv_view(cache, &kv)) return bad(c, msg);
  const size_t es = dtype_bytes(dtype);
  if (!es) return bad(c, "kv attention: unknown row type");
  if (n == 0) return MXQ_OK;
  if (!q || !table || !ctx_len || !cu || !out) return bad(c, "kv attention: null pointer");
  if (n_req == 0 || n_req > MXQ_KV_MAX_REQUESTS) return bad(c, "kv attention: 1 to 8192 requests");
  if (n_heads == 0 || n_heads > 4096 || n_heads % (size_t)kv.heads)
    return bad(c, "kv attention: the query heads are a multiple of the cache's heads");
  if (max_pages == 0 || max_pages > (1u << 26)) return bad(c, "kv attention: bad block table width");
  if (n > (1u << 24) || max_new == 0) return bad(c, "kv attention: bad number of rows");
  if (!(scale == scale)) return bad(c, "kv attention: the scale is NaN");
  if (q_stride < n_heads * (size_t)kv.dim) return bad(c, "kv attention: rows overlap");
  if (!aligned16(q) || !aligned16(out) || q_stride * es % 16)
    return bad(c, "kv attention: rows must start on 16-byte boundaries");
  ServeDevice g(ctx_device(c));
  ServeWs ws;
  if (int rc = ctx_serve_ws(c, &ws)) return rc;
  AttnArgs a{};
  a.c = kv;
  a.q = q;
  a.out = out;
  a.lse = lse;
  a.table = table;
  a.ctx_len = ctx_len;
  a.cu = cu;
  a.q_stride = (long)q_stride;
  a.dtype = dtype;
  a.R = (int)n_req;
  a.n = (int)n;
  a.Hq = (int)n_heads;
  a.G = (int)(n_heads / kv.heads);
  a.max_pages = (int)max_pages;
  a.scale2 = scale * 1.44269504088896341f;
  a.counters = ws.counters + 1;
  a.part = reinterpret_cast<float*>(ws.scratch);
  int ctas = 2 * ws.sms;
  const int fit = (int)(kServeScratch / (2 * kMaxRows * (size_t)(kv.dim + 2) * 4));
  if (ctas > fit) ctas = fit;
  if (ctas > (int)kServeCounters - 1) ctas = (int)kServeCounters - 1;
  // eight rows a tile while no request has more (16-row tiles spend twice the
  // registers and, below nine rows, the same MMAs)
  const bool two = max_new * (size_t)a.G > 8;
  const cudaStream_t st = ctx_stream(c);
  const bool f32 = dtype == MXQ_DT_F32;
  const cudaError_t e = kv.dim == 64 ? launch_d<64>(a, two, f32, ctas, st) : launch_d<128>(a, two, f32, ctas, st);
  return serve_launched(c, e, "kv attention");
}

}  // extern "C"
