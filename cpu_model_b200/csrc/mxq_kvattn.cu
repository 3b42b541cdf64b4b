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
// The query takes three digits (2^-23 of its largest element), the probabilities
// two for 16-bit rows (2^-16 of the block's largest, a 128th of bf16's
// rounding of the result) and three for fp32 rows.  Lengths, maxima, sums and O
// are fp32.
//
// Fragments: B's columns are tokens (S) and dimensions (O).  The order of the
// summed index is free as long as A and B agree, so K rows are read 16 bytes a
// lane as stored, V was stored in the order in which S leaves its
// probabilities (eight tokens a lane), and nothing is shuffled.
//
// Work: units (request, head, tile of query rows), each as many places long
// as it has blocks and kStart more, laid out in one line that is cut into equal
// pieces, one a warp, whatever the lengths are; every CTA finds its pieces by
// summing the lengths itself.  A warp runs through its piece with one ring of
// cp.async stages that does not stop at a unit's end.  Units that lie in one
// piece are written by its warp; those cut by a piece's end are joined by the
// CTA when its warps are done, and those cut by a CTA's end by the last of
// their CTAs, from workspace, in the order of the pieces, so the result
// does not depend on who was last.
//
// Bound by HBM while there are many blocks, by latency else.  32 requests of 2.2k
// tokens, 32 heads of 128, fp32 rows: 117 us, 4.85 TB/s of cache (74 % of a copy).
// 192 requests of 16 to 8191 tokens, 32 heads over 8, bf16: 123 us, 4.6 TB/s; the
// starts of so many units are the rest.  Two requests of 100k to 131k tokens, 16
// heads over 2 of 64, fp16: 22 us, 2.6 TB/s; the chain length -> page -> scale and K
// before a piece's first block, and the join, take two thirds of it.  One request of
// 517 tokens, 32 heads, fp32: 9.3 us, that chain and nothing else.  At D = 128 the
// tiles of one and of eight rows spill 42 to 226 bytes a thread at the 168
// registers that 12 warps leave them; what that costs has not been measured.
#include "mxq_serve.cuh"

namespace mxq {

namespace {

constexpr int kMaxRows = 16;             // query rows a unit
constexpr int kStages = 2;               // blocks a warp has in its ring
// Places a unit's start takes: what its rows, their end and the join cost, in
// blocks (192 unequal requests: 132 us with 1, 126 with 2, 121 with 4, 123 with 10).
constexpr int kStart = 4;
constexpr int kMinPiece = 1;             // places a piece at least
constexpr int kWholeBlocks = 3;          // blocks a warp of a unit that a CTA keeps to itself, at most
constexpr size_t kPromptUnits = 32;      // units of the prompts' kernel that are worth it

struct AttnArgs {
  KvView c;
  const void* q;
  void* out;
  float* lse;
  const int32_t *table, *ctx_len, *cu;
  long q_stride;
  int dtype, R, n, Hq, G, max_pages;
  int few;                               // requests with more rows a K/V head are another kernel's
  float scale2;                          // scale * log2(e)
  uint32_t* counters;                    // [CTAs], zero
  float* warp_part;                      // [CTAs * warps][rows][D + 2]
  float* cta_part;                       // [CTAs][2][rows][D + 2]
};

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

// a / b for a >= 0, b > 0: lengths almost always fit 32 bits, where a division
// is a fifth of the instructions.
__device__ __forceinline__ long div_long(long a, long b) {
  if (((a | b) >> 32) == 0) return (long)((uint32_t)a / (uint32_t)b);
  return a / b;
}

// Start of request r's rows (r = R: their end), inside q whatever is given.
__device__ __forceinline__ int row_start(const AttnArgs& a, int r) { return min(max(a.cu[r], 0), a.n); }

// Rows [0, nrows) of a tile: row i is query head head * G + (tile's row) % G of
// token row0 + (tile's row) / G.
template <int D>
__device__ __forceinline__ void write_row(const AttnArgs& a, int row0, int first, int row, int head, int d,
                                          const float (&o)[4], float m, float l) {
  const int gr = first + row, t = gr / a.G, h = head * a.G + (gr - t * a.G);
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const float y[4] = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
  const long at = (long)(row0 + t) * a.Hq + h;
  store4_dt(a.dtype, a.out, at * D + d, y);
  if (a.lse && d == 0) a.lse[at] = l == 0.0f ? neg_inf() : m * kLn2 + logf(l);
}

// ------------------------------------------------------------------ tiles --
// A tile is a warp's query rows of one unit: its digits, running maxima and sums,
// and O.  start() takes the rows, keys() a block's K (leaving the
// probabilities), values() its V, park() puts (O, maxima, sums) where another may
// join them, write() the finished rows where they belong.

// Digits of four fixed-point numbers, a byte of a word each; digit 0 is the uppermost.
__device__ __forceinline__ void digits3(const float (&x)[4], float inv, bool finite, uint32_t (&dig)[3]) {
  dig[0] = dig[1] = dig[2] = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    int q = finite ? __float2int_rn(x[e] * inv) : 0;
#pragma unroll
    for (int p = 2; p >= 0; --p) {
      dig[p] |= (uint32_t)(q & 0xFF) << (8 * e);
      q = (q + 128) >> 8;
    }
  }
}

// The step 2^ex of a row whose largest element has the bits `top`: |q| <=
// 127 * 256^2; tiny rows keep a step that is a normal number.
struct Step {
  bool finite;
  float inv, scale;                      // 2^-ex, 2^ex scale log2(e)
  __device__ __forceinline__ Step(uint32_t top, float scale2) {
    finite = top < 0x7f800000u;
    const int ex = max(e8m0_exponent<127>(__uint_as_float(top)) - 16, -126);
    inv = finite ? __int_as_float((127 - ex) << 23) : 0.0f;
    scale = finite ? __int_as_float((ex + 127) << 23) * scale2 : __int_as_float(0x7fc00000);
  }
};

// A block's maximum joined to a row's running one: what O and the sum are
// to be multiplied with (alpha), the block's weight (beta), and what to
// subtract from the block's scores.
struct Rise {
  float alpha, beta, base;
  bool none;                             // no key of the block is seen
  __device__ __forceinline__ Rise(float& mx, float bm) {
    none = bm == neg_inf();
    const float mn = fmaxf(mx, bm), ms = mn == neg_inf() ? 0.0f : mn;
    beta = none ? 0.0f : ex2(bm - ms);
    alpha = ex2(mx - ms);
    base = none ? 0.0f : bm;
    mx = mn;
  }
};

template <int NP>
struct Top {                             // what probability 1 is in fixed point, 127 * 256^(NP-1)
  static constexpr float k = NP == 2 ? 32512.0f : 8323072.0f;
};

// Rows of a unit in the MMA's layout: 8 or 16 of them (16 where a unit has more
// than 8, so that a block is read half as often).
template <int D_, int MT, int NP, int W>
struct MmaTile {
  static constexpr int D = D_;
  static constexpr int kRows = 8 * MT;
  static constexpr int kWarps = W;
  static constexpr int kJ = D / 64;                       // 64-dimension halves
  static constexpr int kU = D / 16;                       // V words of 16 dimensions
  static constexpr int kTiles = MT == 1 ? 2 : 3;          // MMA row tiles of S: upper digits of 8 rows each, then the lowest
  static constexpr int kTilesP = NP == 2 ? MT : kTiles;   // of O

  uint32_t qa[MT][3][kJ][4];
  float qs[MT];
  int last[MT];
  float o[MT][kU][4];
  float mx[MT], sum[MT];
  uint32_t pa[MT][NP][2];                // probabilities' digits, slots 0-3 and 4-7
  float fac[MT];

  // Place of a 16-byte piece of K / V in the ring: K rows of 128 bytes have
  // every other row's halves exchanged, so that a quarter warp's two rows lie in
  // different banks.
  static __device__ __forceinline__ int k_place(int ch) { return D == 128 ? ch ^ ((ch >> 3 & 1) << 2) : ch; }
  static __device__ __forceinline__ int v_place(int ch) { return ch; }

  // A fragments: 64 dimensions are two k-steps; lane (r8, c4) has 16 values of
  // row r8: words 0, 1 of step 0 and 2, 3 of step 1.
  __device__ __forceinline__ void start(const AttnArgs& a, int row0, int tile, int head, int nrows, int past) {
    const int lane = threadIdx.x & 31, c4 = lane & 3, r8 = lane >> 2;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int row = m * 8 + r8, gr = tile * kRows + row, t = gr / a.G, h = head * a.G + (gr - t * a.G);
      float x[kJ][4][4];
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < kJ; ++j)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
#pragma unroll
          for (int e = 0; e < 4; ++e) x[j][w][e] = 0.0f;
          if (row < nrows)
            load4_dt(a.dtype, a.q, (long)(row0 + t) * a.q_stride + (long)h * D + j * 64 + c4 * 16 + w * 4, x[j][w]);
#pragma unroll
          for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(x[j][w][e]) & 0x7fffffffu);
        }
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const Step st(top, a.scale2);
#pragma unroll
      for (int j = 0; j < kJ; ++j)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          uint32_t dig[3];
          digits3(x[j][w], st.inv, st.finite, dig);
#pragma unroll
          for (int p = 0; p < 3; ++p) qa[m][p][j][w] = dig[p];
        }
      qs[m] = st.scale;
      last[m] = row < nrows ? past + t : -1;
      mx[m] = neg_inf();
      sum[m] = 0.0f;
#pragma unroll
      for (int u = 0; u < kU; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[m][u][e] = 0.0f;
    }
  }

  __device__ __forceinline__ void keys(const uint8_t* k, int key0, float ks, float vs, uint8_t*) {
    const int lane = threadIdx.x & 31, c4 = lane & 3, r8 = lane >> 2;
    int acc[kTiles][4][4];
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[t][n][e] = 0;
#pragma unroll
    for (int j = 0; j < kJ; ++j)
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const int row = 8 * n + r8;
        const int ch = D == 128 ? row * 8 + ((j * 4 + c4) ^ ((row & 1) << 2)) : row * 4 + c4;
        const uint4 b = *reinterpret_cast<const uint4*>(k + ch * 16);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          mma_s8(acc[m][n], qa[m][0][j][0], qa[m][1][j][0], qa[m][0][j][1], qa[m][1][j][1], b.x, b.y);
          mma_s8(acc[m][n], qa[m][0][j][2], qa[m][1][j][2], qa[m][0][j][3], qa[m][1][j][3], b.z, b.w);
        }
        mma_s8(acc[kTiles - 1][n], qa[0][2][j][0], MT == 2 ? qa[MT - 1][2][j][0] : 0u, qa[0][2][j][1],
               MT == 2 ? qa[MT - 1][2][j][1] : 0u, b.x, b.y);
        mma_s8(acc[kTiles - 1][n], qa[0][2][j][2], MT == 2 ? qa[MT - 1][2][j][2] : 0u, qa[0][2][j][3],
               MT == 2 ? qa[MT - 1][2][j][3] : 0u, b.z, b.w);
      }
    float alpha[MT];
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
          const float s = fmaf((float)hl, 256.0f, (float)acc[kTiles - 1][n][2 * m + e]);
          x[2 * n + e] = key0 + 2 * c4 + 8 * n + e <= last[m] ? s * f : neg_inf();
          bm = fmaxf(bm, x[2 * n + e]);
        }
      bm = fmaxf(bm, __shfl_xor_sync(0xffffffffu, bm, 1));
      bm = fmaxf(bm, __shfl_xor_sync(0xffffffffu, bm, 2));
      const float was = mx[m];
      const Rise r(mx[m], bm);
      alpha[m] = r.alpha;
      same = same && was == mx[m];
      float ps = 0.0f;
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p = ex2(x[4 * g + e] - r.base);
          ps += p;
          // the sum with 2^23 leaves the nearest integer in the low bits
          w[e] = __float_as_uint(fmaf(p, Top<NP>::k, 8388608.0f));
        }
#pragma unroll
        for (int p = NP - 1; p >= 0; --p) {
          pa[m][p][g] = __byte_perm(__byte_perm(w[0], w[1], 0x0040), __byte_perm(w[2], w[3], 0x0040), 0x5410);
          if (p) {
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = (w[e] + 128) >> 8;
          }
        }
      }
      sum[m] = sum[m] * r.alpha + ps * r.beta;
      fac[m] = r.none ? 0.0f : r.beta * vs * (1.0f / Top<NP>::k);
    }
    if (!__all_sync(0xffffffffu, same)) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int u = 0; u < kU; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[m][u][e] *= alpha[m];
    }
  }

  __device__ __forceinline__ void values(const uint8_t* v, const uint8_t*) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const uint4 b = *reinterpret_cast<const uint4*>(v + (u * 32 + lane) * 16);
#pragma unroll
      for (int d = 0; d < 2; ++d) {
        const uint32_t b_lo = d ? b.z : b.x, b_hi = d ? b.w : b.y;
        int pv[kTilesP][4];
#pragma unroll
        for (int t = 0; t < kTilesP; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) pv[t][e] = 0;
#pragma unroll
        for (int m = 0; m < MT; ++m)
          mma_s8(pv[m], pa[m][0][0], pa[m][1][0], pa[m][0][1], pa[m][1][1], b_lo, b_hi);
        if (NP == 3)
          mma_s8(pv[kTilesP - 1], pa[0][NP - 1][0], MT == 2 ? pa[MT - 1][NP - 1][0] : 0u, pa[0][NP - 1][1],
                 MT == 2 ? pa[MT - 1][NP - 1][1] : 0u, b_lo, b_hi);
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float s = (float)(pv[m][e] * 256 + pv[m][2 + e]);
            if (NP == 3) s = fmaf(s, 256.0f, (float)pv[kTilesP - 1][2 * m + e]);
            o[m][u][2 * e + d] = fmaf(s, fac[m], o[m][u][2 * e + d]);
          }
      }
    }
  }

  __device__ __forceinline__ void finish() {
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      sum[m] += __shfl_xor_sync(0xffffffffu, sum[m], 1);
      sum[m] += __shfl_xor_sync(0xffffffffu, sum[m], 2);
    }
  }
  // lane (r8, c4) has dimensions 16 u + 4 c4 .. + 3 of its rows
  __device__ __forceinline__ void write(const AttnArgs& a, int row0, int tile, int head, int nrows) const {
    const int lane = threadIdx.x & 31, c4 = lane & 3, r8 = lane >> 2;
#pragma unroll
    for (int m = 0; m < MT; ++m)
      if (m * 8 + r8 < nrows)
#pragma unroll
        for (int u = 0; u < kU; ++u)
          write_row<D>(a, row0, tile * kRows, m * 8 + r8, head, u * 16 + c4 * 4, o[m][u], mx[m], sum[m]);
  }
  __device__ __forceinline__ void park(float* at, int nrows) const {
    const int lane = threadIdx.x & 31, c4 = lane & 3, r8 = lane >> 2;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int row = m * 8 + r8;
      if (row >= nrows) continue;
#pragma unroll
      for (int u = 0; u < kU; ++u)
        *reinterpret_cast<float4*>(at + row * D + u * 16 + c4 * 4) = make_float4(o[m][u][0], o[m][u][1], o[m][u][2], o[m][u][3]);
      if (c4 == 0) {
        at[kRows * D + row] = mx[m];
        at[kRows * (D + 1) + row] = sum[m];
      }
    }
  }
};

// One query row a unit (a token of a head of its own).  The MMA would leave
// seven of its eight rows empty; dp4a takes the same digits with a lane for each
// token (S, no sums across lanes) and a lane for every D / 32 dimensions (O): under half
// the instructions.
template <int D_, int NP, int W>
struct DotTile {
  static constexpr int D = D_;
  static constexpr int kRows = 1;
  static constexpr int kWarps = W;
  static constexpr int kW = D / 4;                        // words of a K row
  static constexpr int kPairs = D / 64;                   // dimension pairs a lane: lane, lane + 32

  uint32_t q[3][kW];                     // the row's digits, the same in every lane
  float qs;
  int last;
  float o[kPairs][2];
  float mx, sum, fac;

  // a quarter warp reads 8 rows, or 8 dimension pairs: their pieces are
  // rotated so that they lie in different banks
  static __device__ __forceinline__ int k_place(int ch) {
    return D == 128 ? ch ^ (ch >> 3 & 7) : ch ^ (ch >> 3 & 3);
  }
  static __device__ __forceinline__ int v_place(int ch) { return ch ^ (ch >> 3 & 3); }

  __device__ __forceinline__ void start(const AttnArgs& a, int row0, int tile, int head, int, int past) {
    const int lane = threadIdx.x & 31;
    const int t = tile / a.G, h = head * a.G + (tile - t * a.G);
    float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    uint32_t top = 0;
    if (lane < D / 4) {
      load4_dt(a.dtype, a.q, (long)(row0 + t) * a.q_stride + (long)h * D + lane * 4, x);
#pragma unroll
      for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
    }
    const Step st(__reduce_max_sync(0xffffffffu, top), a.scale2);
    uint32_t dig[3];
    digits3(x, st.inv, st.finite, dig);
#pragma unroll
    for (int p = 0; p < 3; ++p)
#pragma unroll
      for (int w = 0; w < kW; ++w) q[p][w] = __shfl_sync(0xffffffffu, dig[p], w);
    qs = st.scale;
    last = past + t;
    mx = neg_inf();
    sum = 0.0f;
#pragma unroll
    for (int u = 0; u < kPairs; ++u) o[u][0] = o[u][1] = 0.0f;
  }

  __device__ __forceinline__ void keys(const uint8_t* k, int key0, float ks, float vs, uint8_t* scratch) {
    const int lane = threadIdx.x & 31;
    int s[3] = {0, 0, 0};
#pragma unroll
    for (int j = 0; j < D / 16; ++j) {
      const uint4 b = *reinterpret_cast<const uint4*>(k + k_place(lane * (D / 16) + j) * 16);
      const uint32_t w[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int p = 0; p < 3; ++p) s[p] = __dp4a((int)w[e], (int)q[p][j * 4 + e], s[p]);
    }
    float x = fmaf((float)(s[0] * 256 + s[1]), 256.0f, (float)s[2]) * (qs * ks);
    if (key0 + lane > last) x = neg_inf();
    // the block's maximum as an integer with the floats' order
    int key = __float_as_int(x);
    key ^= (key >> 31) & 0x7fffffff;
    key = __reduce_max_sync(0xffffffffu, key);
    const Rise r(mx, __int_as_float(key ^ ((key >> 31) & 0x7fffffff)));
    const float p = ex2(x - r.base);
    sum = sum * r.alpha + p * r.beta;
    fac = r.none ? 0.0f : r.beta * vs * (1.0f / Top<NP>::k);
#pragma unroll
    for (int u = 0; u < kPairs; ++u) {
      o[u][0] *= r.alpha;
      o[u][1] *= r.alpha;
    }
    // the token's digits where V's words have its byte: token 8 j + 2 c + b is byte 2 (j % 2) + b of word 2 c + j / 2
    uint32_t v = __float_as_uint(fmaf(p, Top<NP>::k, 8388608.0f));
    const int at = ((lane >> 1) & 3) * 8 + (lane >> 4) * 4 + ((lane >> 3) & 1) * 2 + (lane & 1);
#pragma unroll
    for (int d = NP - 1; d >= 0; --d) {
      scratch[d * 32 + at] = (uint8_t)v;
      v = (v + 128) >> 8;
    }
    __syncwarp();
  }

  __device__ __forceinline__ void values(const uint8_t* v, const uint8_t* scratch) {
    const int lane = threadIdx.x & 31;
    int s[kPairs][2][NP];
#pragma unroll
    for (int u = 0; u < kPairs; ++u)
#pragma unroll
      for (int d = 0; d < 2; ++d)
#pragma unroll
        for (int p = 0; p < NP; ++p) s[u][d][p] = 0;
#pragma unroll
    for (int c = 0; c < 4; c += 2) {
      uint32_t pw[NP][4];                // words of eight-token groups c and c + 1
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        const uint4 w = *reinterpret_cast<const uint4*>(scratch + p * 32 + c * 8);
        pw[p][0] = w.x; pw[p][1] = w.y; pw[p][2] = w.z; pw[p][3] = w.w;
      }
#pragma unroll
      for (int u = 0; u < kPairs; ++u)
#pragma unroll
        for (int cc = 0; cc < 2; ++cc) {
          const uint4 b = *reinterpret_cast<const uint4*>(v + v_place((lane + 32 * u) * 4 + c + cc) * 16);
#pragma unroll
          for (int p = 0; p < NP; ++p) {
            s[u][0][p] = __dp4a((int)b.x, (int)pw[p][2 * cc], s[u][0][p]);
            s[u][0][p] = __dp4a((int)b.y, (int)pw[p][2 * cc + 1], s[u][0][p]);
            s[u][1][p] = __dp4a((int)b.z, (int)pw[p][2 * cc], s[u][1][p]);
            s[u][1][p] = __dp4a((int)b.w, (int)pw[p][2 * cc + 1], s[u][1][p]);
          }
        }
    }
#pragma unroll
    for (int u = 0; u < kPairs; ++u)
#pragma unroll
      for (int d = 0; d < 2; ++d) {
        float y = (float)(s[u][d][0] * 256 + s[u][d][1]);
        if (NP == 3) y = fmaf(y, 256.0f, (float)s[u][d][NP - 1]);
        o[u][d] = fmaf(y, fac, o[u][d]);
      }
  }

  __device__ __forceinline__ void finish() {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
  __device__ __forceinline__ void write(const AttnArgs& a, int row0, int tile, int head, int) const {
    const int lane = threadIdx.x & 31;
    const int t = tile / a.G, h = head * a.G + (tile - t * a.G);
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    const long at = (long)(row0 + t) * a.Hq + h;
#pragma unroll
    for (int u = 0; u < kPairs; ++u) store2_dt(a.dtype, a.out, at * D + 64 * u + 2 * lane, o[u][0] * inv, o[u][1] * inv);
    if (a.lse && lane == 0) a.lse[at] = sum == 0.0f ? neg_inf() : mx * kLn2 + logf(sum);
  }
  __device__ __forceinline__ void park(float* at, int) const {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int u = 0; u < kPairs; ++u) *reinterpret_cast<float2*>(at + 64 * u + 2 * lane) = make_float2(o[u][0], o[u][1]);
    if (lane == 0) {
      at[D] = mx;
      at[D + 1] = sum;
    }
  }
};

// A piece's share of a unit that other pieces share too.
struct Part {
  long unit0;                            // the unit's place in the line
  float* at;                             // [rows][D], maxima [rows], sums [rows]
  int row0, tile, head, nrows;           // rows: tile * kRows + 0 .. nrows - 1 of the request that starts at row0
  int g_first, g_last;                   // the pieces that share it
  int valid;
};

// A running softmax (m, l, y) joined with another.
__device__ __forceinline__ void join(float& m, float& l, float (&y)[4], float pm, float pl, const float4& v) {
  const float mn = fmaxf(m, pm), ms = mn == neg_inf() ? 0.0f : mn;
  const float fa = ex2(m - ms), fb = ex2(pm - ms);
  l = l * fa + pl * fb;
  y[0] = y[0] * fa + v.x * fb;
  y[1] = y[1] * fa + v.y * fb;
  y[2] = y[2] * fa + v.z * fb;
  y[3] = y[3] * fa + v.w * fb;
  m = mn;
}

template <typename Tile>
__global__ void __launch_bounds__(Tile::kWarps * 32, 1) kv_attn_kernel(AttnArgs a) {
  constexpr int D = Tile::D, kRows = Tile::kRows, kWarps = Tile::kWarps, kThreads = kWarps * 32;
  constexpr int kPart = (kRows * (D + 2) + 3) / 4 * 4;   // floats of a part, whole 16-byte pieces
  constexpr int kStage = 64 * D;                   // one block's K and V
  static_assert(kPart * 4 <= kStages * kStage, "a part takes its warp's ring");
  static_assert(kWarps * kPart <= 8 * kMaxRows * (D + 2) && kPart <= kMaxRows * (D + 2), "parts take their place in the workspace");
  extern __shared__ __align__(16) uint8_t sm[];
  uint8_t* scratch = sm + kWarps * kStages * kStage + (threadIdx.x >> 5) * 128;   // a tile's own
  long* s_sum = reinterpret_cast<long*>(sm + kWarps * (kStages * kStage + 128));  // [R + 1]
  __shared__ long s_warp[kWarps];
  __shared__ Part s_part[kWarps * 2];
  __shared__ int s_flag;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int Hkv = a.c.heads, G = a.G, nb = a.c.nb;

  // ---- the line of work: units * places of every request, summed.  A warp's
  // worth of requests is summed by every warp for itself, without a barrier.
  auto blocks_of = [&](int ctx) { return ceil_div(table_keys(a.c, a.max_pages, ctx), 32); };
  auto units_of = [&](int r, int* blocks) {
    *blocks = 0;
    if (r >= a.R) return 0;
    const int rows = (row_start(a, r + 1) - row_start(a, r)) * G, len = a.ctx_len[r];
    if (rows <= 0 || rows > a.few || len <= 0) return 0;
    *blocks = blocks_of(len);
    return (rows + kRows - 1) / kRows * Hkv;
  };
  if (lane < 2) s_part[warp * 2 + lane].valid = 0;
  const int pieces = gridDim.x * kWarps, piece = blockIdx.x * kWarps + warp;
  long lo, hi, len;
  int share = 0;                         // a unit a CTA: blocks of it a warp
  if (a.R <= 32) {
    int blocks;
    const int u = units_of(lane, &blocks), most = __reduce_max_sync(0xffffffffu, blocks);
    const long w = (long)u * (blocks + kStart);
    long sum = w;
    int units = u;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long x = __shfl_up_sync(0xffffffffu, sum, o);
      const int y = __shfl_up_sync(0xffffffffu, units, o);
      if (lane >= o) sum += x, units += y;
    }
    if (lane < a.R) s_sum[lane] = sum - w;           // every warp writes the same
    const long total = __shfl_sync(0xffffffffu, sum, 31);
    if (lane == 0) s_sum[a.R] = total;
    __syncwarp();
    // Few short units: a CTA each, its blocks shared out over the warps, and
    // nothing to join outside it.  (At 36 blocks the SM that has them all takes as
    // long as several would with the join through workspace, 4500 cycles.)
    if (__shfl_sync(0xffffffffu, units, 31) <= (int)gridDim.x && most <= kWholeBlocks * kWarps) {
      const uint32_t before = __ballot_sync(0xffffffffu, units <= (int)blockIdx.x);
      const int r = __popc(before);                  // the request of this CTA's unit
      if (r >= 32) {
        lo = hi = 0;
        len = 1;
      } else {
        const int nblk = __shfl_sync(0xffffffffu, blocks, r);
        const int in = (int)blockIdx.x - __shfl_sync(0xffffffffu, units - u, r);
        const long unit0 = __shfl_sync(0xffffffffu, sum - w, r) + (long)in * (nblk + kStart);
        share = max(1, (nblk + kWarps - 1) / kWarps);
        lo = unit0 + kStart + warp * share;
        hi = min(lo + share, unit0 + kStart + nblk);
        len = 1;
      }
    } else {
      len = max(div_long(total + pieces - 1, pieces), (long)kMinPiece);
      lo = piece * len;
      hi = min(lo + len, total);
    }
  } else {
    long base = 0;
    for (int r0 = 0; r0 < a.R; r0 += kThreads) {
      int blocks;
      const int u = units_of(r0 + tid, &blocks);
      const long w = (long)u * (blocks + kStart);
      long sum = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long x = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += x;
      }
      __syncthreads();
      if (lane == 31) s_warp[warp] = sum;
      __syncthreads();
      long before = base;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) {
        if (i < warp) before += s_warp[i];
        base += s_warp[i];
      }
      if (r0 + tid < a.R) s_sum[r0 + tid] = before + sum - w;
    }
    if (tid == 0) s_sum[a.R] = base;
    __syncthreads();
    len = max(div_long(base + pieces - 1, pieces), (long)kMinPiece);
    lo = piece * len;
    hi = min(lo + len, base);
  }

  uint8_t* ring = sm + warp * (kStages * kStage);
  const uint32_t ring_s = smem_u32(ring);

  auto request_of = [&](long pos) {      // the request with work at a place of the line
    int x = 0, y = a.R;
    while (y - x > 1) {
      const int mid = (x + y) >> 1;
      if (s_sum[mid] <= pos) x = mid;
      else y = mid;
    }
    return x;
  };

  // ---- places pos + lane: the page of the block there (look), and then where
  // it is in the cache (seen; -1: a page that holds no keys, no block, or one that no
  // row of the tile sees)
  long place = -1;
  int page = -1, page_head = 0, page_sub = 0;
  auto look = [&](long pos) {
    pos += lane;
    page = -1;
    if (pos < hi) {
      const int r = request_of(pos);
      const int row0 = row_start(a, r), rows = (row_start(a, r + 1) - row0) * G, ctx = a.ctx_len[r];
      const int per = blocks_of(ctx) + kStart, tiles = (rows + kRows - 1) / kRows;
      const long in = pos - s_sum[r];
      const int unit = (int)div_long(in, per), b = (int)(in - (long)unit * per) - kStart;
      const int head = unit / tiles, tile = unit - head * tiles;
      const int last_row = min((tile + 1) * kRows, rows) - 1;
      const int sees = ctx - rows / G + last_row / G + 1;
      const int pg = b / nb;
      page_head = head;
      page_sub = b - pg * nb;
      if (b >= 0 && b * 32 < sees && pg < a.max_pages) page = a.table[(long)r * a.max_pages + pg];
    }
  };
  auto seen = [&]() { place = page >= 0 && page < a.c.n_pages ? kv_block(a.c, page, page_head, page_sub) : -1; };
  const int mine = lo < hi ? (int)(hi - lo) : 0;
  // The ring holds the next two blocks (places without one are passed over):
  // where in the piece they are, their scales, and where in the cache.  K and V
  // are groups of their own, so that K's part of a stage is refilled while V's
  // is still in use.
  int to_see = 0;                        // first place that has not been looked at
  int q_pos0 = -1, q_pos1 = -1;
  uint32_t q_ks0 = 0, q_ks1 = 0, q_vs0 = 0, q_vs1 = 0;
  long q_at0 = 0, q_at1 = 0;
  auto fetch_k = [&](int s) {
    int found = -1;
    while (to_see < mine) {
      if ((to_see & 31) == 0 && to_see) {
        look(lo + to_see);
        seen();
      }
      const uint32_t here = __ballot_sync(0xffffffffu, place >= 0) >> (to_see & 31);
      if (here) {
        found = to_see + __ffs((int)here) - 1;
        to_see = found + 1;
        break;
      }
      to_see = (to_see | 31) + 1;
    }
    if (s) q_pos1 = found;
    else q_pos0 = found;
    if (found >= 0) {
      const long at = __shfl_sync(0xffffffffu, place, found & 31);
      if (s) q_at1 = at, q_ks1 = a.c.ks[at], q_vs1 = a.c.vs[at];
      else q_at0 = at, q_ks0 = a.c.ks[at], q_vs0 = a.c.vs[at];
      const int8_t* src = a.c.k + at * (32 * D);
#pragma unroll
      for (int u = 0; u < 2 * D / 32; ++u)
        cp16(ring_s + s * kStage + Tile::k_place(u * 32 + lane) * 16, src + (u * 32 + lane) * 16);
    }
    cp_commit();
  };
  auto fetch_v = [&](int s) {
    if ((s ? q_pos1 : q_pos0) >= 0) {
      const int8_t* src = a.c.v + (s ? q_at1 : q_at0) * (32 * D);
#pragma unroll
      for (int u = 0; u < 2 * D / 32; ++u)
        cp16(ring_s + s * kStage + 32 * D + Tile::v_place(u * 32 + lane) * 16, src + (u * 32 + lane) * 16);
    }
    cp_commit();
  };
  int stage = 0;                         // of the next block

  // ---- the unit at place i of the piece
  int req = 0, row0 = 0, tile = 0, head = 0, nrows = 0, past = 0, end = 0, g_first = 0, g_last = 0;
  long unit0 = 0;
  bool has = false;                      // the piece has blocks of it to attend to (or all it has: none)
  auto unit_at = [&](int i) {
    const long pos = lo + i;
    while (s_sum[req + 1] <= pos) ++req;
    row0 = row_start(a, req);
    const int rows = (row_start(a, req + 1) - row0) * G, ctx = a.ctx_len[req];
    const int per = blocks_of(ctx) + kStart, tiles = (rows + kRows - 1) / kRows;
    const long in = pos - s_sum[req];
    const int unit = (int)div_long(in, per), skip = (int)(in - (long)unit * per);
    head = unit / tiles;
    tile = unit - head * tiles;
    unit0 = pos - skip;
    end = (int)min((long)mine, (long)i + per - skip);          // this piece's places of the unit: i .. end - 1
    nrows = min(kRows, rows - tile * kRows);
    past = ctx - rows / G;
    // blocks with keys that the tile's last row sees
    const int blocks = blocks_of(min(ctx, past + (tile * kRows + nrows - 1) / G + 1));
    // the pieces with blocks of it
    if (share) {
      g_first = blockIdx.x * kWarps;
      g_last = g_first + max(blocks - 1, 0) / share;
    } else {
      g_first = (int)div_long(unit0 + kStart, len);
      g_last = blocks ? (int)div_long(unit0 + kStart + blocks - 1, len) : g_first;
    }
    has = blocks ? skip < kStart + blocks && skip + (end - i) > kStart
                 : skip <= kStart && skip + (end - i) > kStart;   // a unit without keys: whoever has its first place
  };
  if (mine) {
    look(lo);                            // the pages are on their way while the unit is worked out
    req = request_of(lo);
    unit_at(0);
    seen();
    fetch_k(0);
    fetch_v(0);
    fetch_k(1);
    fetch_v(1);
  }
  for (int i = 0; i < mine;) {
    if (i) unit_at(i);
    Tile t;
    if (has) t.start(a, row0, tile, head, nrows, past);
    i = end;
    for (;;) {
      const int at = stage ? q_pos1 : q_pos0;
      if (at < 0 || at >= end) break;
      uint8_t* st = ring + stage * kStage;
      const uint32_t ks = stage ? q_ks1 : q_ks0, vs = stage ? q_vs1 : q_vs0;
      cp_wait<2 * kStages - 1>();        // K is there; V and what follows may be on the way
      __syncwarp();
      t.keys(st, ((int)(lo + at - unit0) - kStart) * 32, e8m0_to_float(ks), e8m0_to_float(vs), scratch);
      __syncwarp();                      // every lane has read it before it is refilled
      fetch_k(stage);
      cp_wait<2 * kStages - 1>();        // V
      __syncwarp();
      t.values(st + 32 * D, scratch);
      __syncwarp();
      fetch_v(stage);
      stage ^= 1;
    }
    if (!has) continue;

    t.finish();
    if (g_first == g_last) {
      t.write(a, row0, tile, head, nrows);
    } else {
      // the piece's last unit may take the ring's place, an earlier one goes to workspace
      const bool final = i >= mine;
      if (final) {
        cp_wait<0>();
        __syncwarp();
      }
      float* at = final ? reinterpret_cast<float*>(ring) : a.warp_part + (long)piece * kPart;
      t.park(at, nrows);
      if (lane == 0) s_part[warp * 2 + (piece == g_first ? 1 : 0)] = Part{unit0, at, row0, tile, head, nrows, g_first, g_last, 1};
    }
  }
  cp_wait<0>();

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
  __syncthreads();                       // every part of this CTA is where its record says

  // ---- the CTA's parts of each cut unit joined, in the order of the pieces:
  // records of one unit follow one another
  static_assert(kWarps * 2 <= 32, "a record a lane");
  const bool valid = lane < kWarps * 2 && s_part[lane].valid;
  const uint32_t all = __ballot_sync(0xffffffffu, valid);
  uint32_t starts;
  {
    const uint32_t below = all & ((1u << lane) - 1);
    const bool first = !below || s_part[31 - __clz(below)].unit0 != s_part[lane < kWarps * 2 ? lane : 0].unit0;
    starts = __ballot_sync(0xffffffffu, valid && first);
  }
  int open[2] = {-1, -1};                // records of the units that go on outside this CTA
  int groups = 0;
  for (; starts; starts &= starts - 1, ++groups) {
    const int g = __ffs((int)starts) - 1;
    const uint32_t rest = starts & (starts - 1);     // the next unit's first record
    const uint32_t group = all & ~((1u << g) - 1) & (rest ? (1u << (__ffs((int)rest) - 1)) - 1 : 0xffffffffu);
    const Part& p = s_part[g];
    const int p_nrows = p.nrows, c_first = p.g_first / kWarps;
    const bool outside = c_first != p.g_last / kWarps;
    const int slot = c_first == (int)blockIdx.x ? 1 : 0;
    if (outside) open[slot] = g;
    float* to = a.cta_part + ((long)blockIdx.x * 2 + slot) * kPart;
    // small units start at different warps
    for (int w = (tid + kThreads - (groups * 32) % kThreads) % kThreads; w < p_nrows * (D / 4); w += kThreads) {
      const int row = w / (D / 4), d = (w - row * (D / 4)) * 4;
      float m = neg_inf(), l = 0.0f;
      float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      for (uint32_t left = group; left;) {           // four parts' loads at a time
        float pm[4], pl[4];
        float4 v[4];
        bool real[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          real[e] = left != 0;
          const float* q = s_part[left ? __ffs((int)left) - 1 : g].at;
          pm[e] = real[e] ? q[kRows * D + row] : neg_inf();
          pl[e] = q[kRows * (D + 1) + row];
          v[e] = *reinterpret_cast<const float4*>(q + row * D + d);
          left &= left - 1;
        }
        const float top = fmaxf(fmaxf(fmaxf(pm[0], pm[1]), fmaxf(pm[2], pm[3])), m), ms = top == neg_inf() ? 0.0f : top;
        const float fa = ex2(m - ms);
        l *= fa;
        y[0] *= fa; y[1] *= fa; y[2] *= fa; y[3] *= fa;
        m = top;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (!real[e]) continue;
          const float f = ex2(pm[e] - ms);
          l += f * pl[e];
          y[0] += f * v[e].x; y[1] += f * v[e].y; y[2] += f * v[e].z; y[3] += f * v[e].w;
        }
      }
      if (!outside) {
        write_row<D>(a, p.row0, p.tile * kRows, row, p.head, d, y, m, l);
      } else {
        *reinterpret_cast<float4*>(to + row * D + d) = make_float4(y[0], y[1], y[2], y[3]);
        if (d == 0) {
          to[kRows * D + row] = m;
          to[kRows * (D + 1) + row] = l;
        }
      }
    }
  }
  if (open[0] < 0 && open[1] < 0) return;          // the same in every thread
  __threadfence();
  for (int s = 0; s < 2; ++s) {
    if (open[s] < 0) continue;
    const Part p = s_part[open[s]];
    const int c_first = p.g_first / kWarps, parts = p.g_last / kWarps - c_first + 1;
    __syncthreads();
    if (tid == 0) {
      // a unit that is cut by a CTA's end is the only one that starts in that CTA and leaves it
      s_flag = atomicAdd(a.counters + c_first, 1u) == (uint32_t)parts - 1;
      if (s_flag) a.counters[c_first] = 0;
    }
    __syncthreads();
    if (!s_flag) continue;
    __threadfence();
    // several threads a result where there are few: each takes every crew-th part
    const int tasks = p.nrows * (D / 4), crew = max(1, min(kThreads / tasks, parts));
    float* s_join = reinterpret_cast<float*>(sm);  // [crew][tasks][6]
    for (int w = tid; w < tasks * crew; w += kThreads) {
      const int who = w / tasks, task = w - who * tasks, row = task / (D / 4), d = (task - row * (D / 4)) * 4;
      float m = neg_inf(), l = 0.0f;
      float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      constexpr int kAhead = 8;
      for (int i = who; i < parts; i += kAhead * crew) {
        float pm[kAhead], pl[kAhead];
        float4 v[kAhead];
#pragma unroll
        for (int e = 0; e < kAhead; ++e) {
          const int at = i + e * crew;
          pm[e] = neg_inf();
          pl[e] = 0.0f;
          v[e] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          if (at < parts) {
            const float* q = a.cta_part + ((long)(c_first + at) * 2 + (at == 0 ? 1 : 0)) * kPart;
            pm[e] = __ldcg(q + kRows * D + row);
            pl[e] = __ldcg(q + kRows * (D + 1) + row);
            v[e] = __ldcg(reinterpret_cast<const float4*>(q + row * D + d));
          }
        }
#pragma unroll
        for (int e = 0; e < kAhead; ++e) join(m, l, y, pm[e], pl[e], v[e]);
      }
      if (crew == 1) {
        write_row<D>(a, p.row0, p.tile * kRows, row, p.head, d, y, m, l);
      } else {
        float* q = s_join + w * 6;
        q[0] = m;
        q[1] = l;
#pragma unroll
        for (int e = 0; e < 4; ++e) q[2 + e] = y[e];
      }
    }
    if (crew > 1) {
      __syncthreads();
      if (tid < tasks) {
        const int row = tid / (D / 4), d = (tid - row * (D / 4)) * 4;
        float m = neg_inf(), l = 0.0f;
        float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int i = 0; i < crew; ++i) {
          const float* q = s_join + (i * tasks + tid) * 6;
          join(m, l, y, q[0], q[1], make_float4(q[2], q[3], q[4], q[5]));
        }
        write_row<D>(a, p.row0, p.tile * kRows, row, p.head, d, y, m, l);
      }
    }
  }
}

// A ring a warp, and the requests' sums.
template <typename Tile>
constexpr size_t attn_smem(size_t requests) {
  return (size_t)Tile::kWarps * (kStages * 64 * Tile::D + 128) + (requests + 1) * 8;
}
constexpr size_t kSmemLimit = 227u << 10, kSmemStatic = 1536;   // of a CTA; what the kernel's own variables may take of it

template <typename Tile>
cudaError_t launch(const AttnArgs& a, int ctas, cudaStream_t st) {
  static SmemAttr attr;
  const size_t smem = attn_smem<Tile>(a.R);
  const cudaError_t e = attr.ensure(kv_attn_kernel<Tile>, smem);
  if (e != cudaSuccess) return e;
  kv_attn_kernel<Tile><<<(unsigned)ctas, Tile::kWarps * 32, smem, st>>>(a);
  return cudaGetLastError();
}

// A tile with 12 warps a CTA, or with 10 where the sums of thousands of
// requests would not fit beside 12 rings (D = 128, from 4096 requests on; 8
// K/V heads, 150 to 350 tokens each, one fp32 row: 4095 requests 426 us, 4096
// 462; four bf16 rows: 455 and 453).
template <template <int> class Tile>
cudaError_t launch_warps(const AttnArgs& a, int ctas, cudaStream_t st) {
  static_assert(attn_smem<Tile<10>>(MXQ_KV_MAX_REQUESTS) + kSmemStatic <= kSmemLimit, "every number of requests fits");
  if constexpr (attn_smem<Tile<12>>(MXQ_KV_MAX_REQUESTS) + kSmemStatic > kSmemLimit)
    if (attn_smem<Tile<12>>(a.R) + kSmemStatic > kSmemLimit) return launch<Tile<10>>(a, ctas, st);
  return launch<Tile<12>>(a, ctas, st);
}
template <int D, int NP> struct Rows {
  template <int W> using One = DotTile<D, NP, W>;
  template <int W> using Eight = MmaTile<D, 1, NP, W>;
  using Sixteen = MmaTile<D, 2, NP, 8>;
  static_assert(attn_smem<Sixteen>(MXQ_KV_MAX_REQUESTS) + kSmemStatic <= kSmemLimit, "every number of requests fits");
};

// One row a unit, eight while no request has more (16-row tiles spend twice the
// registers on them), else sixteen.
template <int D, int NP>
cudaError_t launch_rows(const AttnArgs& a, size_t rows, int ctas, cudaStream_t st) {
  if (rows == 1) return launch_warps<Rows<D, NP>::template One>(a, ctas, st);
  if (rows <= 8) return launch_warps<Rows<D, NP>::template Eight>(a, ctas, st);
  return launch<typename Rows<D, NP>::Sixteen>(a, ctas, st);
}
template <int D>
cudaError_t launch_rows(const AttnArgs& a, size_t rows, bool f32, int ctas, cudaStream_t st) {
  return f32 ? launch_rows<D, 3>(a, rows, ctas, st) : launch_rows<D, 2>(a, rows, ctas, st);
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
  a.scale2 = scale * kLog2e;
  a.counters = ws.counters + 1;
  // a part for each warp (12 of up to 8 rows, or 8 of 16) and two for each CTA
  const size_t row = (size_t)(kv.dim + 2) * 4, warp_parts = 8 * kMaxRows * row;
  int ctas = ws.sms;
  const int fit = (int)(kServeScratch / (warp_parts + 2 * kMaxRows * row));
  if (ctas > fit) ctas = fit;
  if (ctas > (int)kServeCounters - 3) ctas = (int)kServeCounters - 3;
  a.warp_part = reinterpret_cast<float*>(ws.scratch);
  a.cta_part = reinterpret_cast<float*>(ws.scratch + (size_t)ctas * warp_parts);
  const size_t rows = max_new * (size_t)a.G;
  a.few = 1 << 30;
  // Prompts' 16-bit rows go to the tensor cores' kernel where the call's rows would
  // fill at least kPromptUnits of its units: one SM with it is as fast as 6 with this
  // one, but its units are not cut along the keys.  The rows of the whole call
  // are counted, since the host does not know whose they are, so a prompt among many
  // single tokens goes there with few units too.  250 decoding requests of 16 to
  // 8191 tokens, 32 heads over 8, bf16: 146 us; with a prompt of 40 rows behind 4000
  // tokens beside them, 8 units, 274 us (fp32 rows, all on this kernel: 207); of 300
  // rows, 40 units, 286 us (321).
  const bool f32 = dtype == MXQ_DT_F32;
  const size_t units = (n * (size_t)a.G + 255) / 256 * kv.heads;
  if (!f32 && rows > kMaxRows && units >= kPromptUnits) {
    a.few = kMaxRows;
    KvPromptArgs p{kv, q, out, lse, table, ctx_len, cu, (long)q_stride, (int)n_req, (int)n, a.Hq, a.G, a.max_pages,
                   kMaxRows, dtype == MXQ_DT_BF16, a.scale2, ws.counters + kServeCounters - 2, ctx_status_word(c)};
    if (int rc = serve_launched(c, launch_kv_prompt(p, ws.sms, ctx_stream(c)), "kv attention of prompts")) return rc;
  }
  const cudaStream_t st = ctx_stream(c);
  const cudaError_t e = kv.dim == 64 ? launch_rows<64>(a, rows, f32, ctas, st) : launch_rows<128>(a, rows, f32, ctas, st);
  return serve_launched(c, e, "kv attention");
}

}  // extern "C"
