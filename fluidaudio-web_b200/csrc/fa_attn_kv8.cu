// Attention over the 8-bit key and value cache (fa_kv8.cuh): out = sum_j p_j v_j / sum_j p_j, p_j = exp(q.k_j - max).
//
// Rows: the G = HQ / H query heads that share a key head times the T queries of a stream, row r = query r / G, head r % G.
//
// Arithmetic.  Codes are whole numbers of 8 bits, so they are exact in f16; the other side of each product is split into an
// f16 value and its f16 residue (22 bits and more) and both go through the same product, so that operands are f32-grade and
// sums are f32.  A query row is scaled by a power of two to [1, 2) before the split and the block's scale multiplies the sums
// afterwards.  Weights are exp(s - the block's own row maximum), so that the largest is 1 whatever the other blocks hold; what
// the block then adds to the running result is scaled by exp(block maximum - running maximum) times the values' scale, in f32.
#include "fa_kv8.cuh"
#include "fa_tc_common.cuh"

#include <type_traits>

namespace {

using kv8::kBlock;
using tc::smem_u32;

constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr float kLog2e = 1.4426950408889634f;

struct AttnParams {
  const float *q;  // query row i of stream s, head h: q + (s*T + i)*ldq + h*HD
  long long ldq;
  const uint8_t *codes;
  const float *lens;  // [S] on the device, or NULL: n for all (complete caches)
  kv8::Rows rows;     // causal: where the queries stand
  int causal, n;
  int S, H, G, T, HD, nblk, vec;
  int rg0, rowgroups; // groups of ROWS rows that this launch takes
  float *out;         // [S*T][H*G*HD]
  __half *y16;        // packed f16 row operand of out (value plane, then residue plane), or NULL
  long long lo_off;
  int R;              // rows of out
  float *pacc, *pml;  // parts of units that several thread blocks share: [grid][2][rows][HDP] and [..][rows][2]
  int *tickets;       // [S*H*rowgroups], zero between launches
  int *status;
  unsigned wait_limit;
};

// What the queries of stream s see: `len` positions at the most, query i limit(i) of them.
struct Sight {
  int start, count, len, causal;
  __device__ __forceinline__ void of(const AttnParams &p, int s, bool &bad) {
    causal = p.causal, bad = false, start = 0, count = p.T, len = p.n;
    if (causal) {
      p.rows.of(s, start, count, bad);
      len = count > 0 ? start + count : 0;
    } else if (p.lens) {
      const float f = p.lens[s];
      bad = !(f >= 0.0f && f <= (float)p.n);
      len = f >= 0.0f ? (int)fminf(f, (float)p.n) : 0;
    }
  }
  __device__ __forceinline__ int limit(int i) const { return !causal ? len : i < count ? start + i + 1 : 0; }
  // a stream of length 0 still has a block that nothing is seen of, so that somebody writes its zeros
  __device__ __forceinline__ int blocks() const { return max(1, (len + kBlock - 1) / kBlock); }
};

__device__ __forceinline__ void mma(float (&c)[4], const uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t h2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *(const uint32_t *)&h;
}
// (a, b) as f16 values, and what they leave as f16 residues
__device__ __forceinline__ void split2(float a, float b, uint32_t &hi, uint32_t &lo) {
  const __half2 h = __floats2half2_rn(a, b);
  const float2 f = __half22float2(h);
  hi = *(const uint32_t *)&h;
  lo = h2(a - f.x, b - f.y);
}
// A word of four codes as two pairs of f16 u - 128.
__device__ __forceinline__ void widen(uint32_t w, uint32_t &b0, uint32_t &b1) {
  const __half2 bias = __half2half2(__ushort_as_half(0x6480));  // 1152
  const uint32_t x = __byte_perm(w, 0x64646464u, 0x4140), y = __byte_perm(w, 0x64646464u, 0x4342);
  const __half2 p = __hsub2(*(const __half2 *)&x, bias), q = __hsub2(*(const __half2 *)&y, bias);
  b0 = *(const uint32_t *)&p, b1 = *(const uint32_t *)&q;
}
// two f32 at once
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpair(uint64_t a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 2^(m - M) for M >= m, 1 where the two are the same infinity
__device__ __forceinline__ float rescale(float m, float M) { return m == M ? 1.0f : ex2(m - M); }

// Query rows are scaled by 2^kUp and weights by about 2^kUpW before they are split (f16 ends at 2^16, and the less of a residue is
// subnormal the better).  What weights are relative to is their block's largest score less kUpW as an f32 has it: where scores
// are so large that the difference is rounded, it is off by at most 8, and it is the reference of the block's sums as well.
constexpr int kUp = 14, kUpW = 7;
constexpr float kScoreUnit = kLog2e / (1 << kUp);  // scores in units of log 2

// Channels 16k + 4t ..+3 of query row `row` for all k, scaled by the power of two that brings its largest element to
// [2^kUp, 2^(kUp+1)); returns 2^kUp over that scale, NaN for a row that is not finite.  The four lanes of a quad hold the row.
template <int KS>
__device__ __forceinline__ float load_row(const AttnParams &p, int s, int h, int row, int t, float (&x)[KS][4]) {
  const int rr = min(row, p.G * p.T - 1), i = rr / p.G;
  const float *qp = p.q + ((long long)s * p.T + i) * p.ldq + (h * p.G + rr - i * p.G) * p.HD;
  uint32_t a = 0;  // largest magnitude, as bits: infinities and NaNs are above all others
#pragma unroll
  for (int k = 0; k < KS; k++) {
    const int d = 16 * k + 4 * t;
    if (p.vec) {
      const float4 v = d < p.HD ? *(const float4 *)(qp + d) : make_float4(0.f, 0.f, 0.f, 0.f);
      x[k][0] = v.x, x[k][1] = v.y, x[k][2] = v.z, x[k][3] = v.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++) x[k][e] = d + e < p.HD ? qp[d + e] : 0.0f;
    }
  }
#pragma unroll
  for (int k = 0; k < KS; k++)
#pragma unroll
    for (int e = 0; e < 4; e++) a = max(a, __float_as_uint(x[k][e]) & 0x7fffffffu);
  a = max(a, __shfl_xor_sync(0xffffffffu, a, 1));
  a = max(a, __shfl_xor_sync(0xffffffffu, a, 2));
  const int bits = (int)(a >> 23), ex = min(max(bits, kUp + 1), 254);
  const float f = __int_as_float((254 + kUp - ex) << 23);
#pragma unroll
  for (int k = 0; k < KS; k++)
#pragma unroll
    for (int e = 0; e < 4; e++) x[k][e] *= f;
  return bits < 255 ? __int_as_float(ex << 23) : __int_as_float(0x7fc00000);
}

// Up to four rows: codes are the ROW operand of the products, 16 positions (or channels) by 16, and the query rows their 8
// columns, 2r the value and 2r + 1 the residue of row r, so that column sums 2t and 2t + 1 meet in one lane: lane (g, t) has
// the scores of row t at the four positions 8 (g/2) + 2j + g%2, and channels 16c + g and 16c + 8 + g of row t's result.
template <int HDP>
struct FewRows {
  static constexpr int ROWS = 4, KS = HDP / 16, PITCH = HDP + 8, RESIDENT = 3;
  uint32_t qb[KS][2];
  float qs, m, l;
  uint64_t o[HDP / 8];  // what the weights' values and their residues gave
  int lim;

  __device__ __forceinline__ void start(const AttnParams &p, int s, int h, int row0, const Sight &sight, int lane) {
    const int g = lane >> 2, t = lane & 3;
    float x[KS][4];
    const float f = load_row<KS>(p, s, h, row0 + (g >> 1), t, x);
    qs = __shfl_sync(0xffffffffu, f, 8 * t);
#pragma unroll
    for (int k = 0; k < KS; k++) {
      uint32_t hi, lo;
      split2(x[k][0], x[k][1], hi, lo);
      qb[k][0] = g & 1 ? lo : hi;
      split2(x[k][2], x[k][3], hi, lo);
      qb[k][1] = g & 1 ? lo : hi;
    }
    lim = row0 + t < p.G * p.T ? sight.limit((row0 + t) / p.G) : sight.len;  // (a row that is not there hinders nobody)
    m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < HDP / 8; i++) o[i] = 0;
  }

  // `all`: every row sees every position of the block
  __device__ __forceinline__ void block(const uint8_t *sb, int first, bool all, int lane) {
    const int g = lane >> 2, t = lane & 3;
    float sc[2][4];
#pragma unroll
    for (int mt = 0; mt < 2; mt++) sc[mt][0] = sc[mt][1] = sc[mt][2] = sc[mt][3] = 0.0f;
    uint32_t w[4 * KS];
#pragma unroll
    for (int c = 0; c < KS; c++) {
      const uint4 w4 = *(const uint4 *)(sb + c * 512 + lane * 16);
      w[4 * c] = w4.x, w[4 * c + 1] = w4.y, w[4 * c + 2] = w4.z, w[4 * c + 3] = w4.w;
    }
#pragma unroll
    for (int mt = 0; mt < 2; mt++)
#pragma unroll
      for (int ks = 0; ks < KS; ks++) {
        uint32_t a0, a1, a2, a3;
        widen(w[2 * mt * KS + ks], a0, a2);
        widen(w[(2 * mt + 1) * KS + ks], a1, a3);
        mma(sc[mt], a0, a1, a2, a3, qb[ks][0], qb[ks][1]);
      }
    const float2 scales = *(const float2 *)(sb + 2 * kBlock * HDP);
    const float f = scales.x * kScoreUnit * qs;
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] = (sc[j >> 1][2 * (j & 1)] + sc[j >> 1][2 * (j & 1) + 1]) * f;
    const int n = lim - first - 8 * (g >> 1) - (g & 1);  // position j of this lane is seen if 2j < n
    if (!all) {
#pragma unroll
      for (int j = 0; j < 4; j++) v[j] = 2 * j < n ? v[j] : -INFINITY;
    }
    float top = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
    const float ref = top - kUpW, M = fmaxf(m, ref), old = rescale(m, M), c = rescale(ref, M), from = ref == -INFINITY ? 0.0f : ref;
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] = ex2(v[j] - from);
    l = fmaf(l, old, ((v[0] + v[1]) + (v[2] + v[3])) * c);
    m = M;
    const float add = lim > first ? c * scales.y : 0.0f;  // (a block that a row sees nothing of may hold NaN)
    const uint64_t add_2 = pair(add, add);
    if (__any_sync(0xffffffffu, old != 1.0f)) {
      const uint64_t old_2 = pair(old, old);
#pragma unroll
      for (int i = 0; i < HDP / 8; i++) o[i] = mul2(o[i], old_2);
    }
    // weights to the lanes that need them as column operand: column g is row g/2's value (g even) or residue, positions 8t..8t+7
    uint32_t hi[2], lo[2], b[2][2];
    split2(v[0], v[1], hi[0], lo[0]);
    split2(v[2], v[3], hi[1], lo[1]);
    const int even = 8 * t + (g >> 1);
#pragma unroll
    for (int kk = 0; kk < 2; kk++) {
      const uint32_t h0 = __shfl_sync(0xffffffffu, hi[kk], even), h1 = __shfl_sync(0xffffffffu, hi[kk], even + 4);
      const uint32_t l0 = __shfl_sync(0xffffffffu, lo[kk], even), l1 = __shfl_sync(0xffffffffu, lo[kk], even + 4);
      const uint32_t x = g & 1 ? l0 : h0, y = g & 1 ? l1 : h1;
      b[kk][0] = __byte_perm(x, y, 0x5410), b[kk][1] = __byte_perm(x, y, 0x7632);
    }
#pragma unroll
    for (int i = 0; i < KS; i++) {
      const uint4 w4 = *(const uint4 *)(sb + kBlock * HDP + i * 512 + lane * 16);
      float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      uint32_t a0, a1, a2, a3;
      widen(w4.x, a0, a2);
      widen(w4.z, a1, a3);
      mma(acc, a0, a1, a2, a3, b[0][0], b[0][1]);
      widen(w4.y, a0, a2);
      widen(w4.w, a1, a3);
      mma(acc, a0, a1, a2, a3, b[1][0], b[1][1]);
      o[2 * i] = fma2(pair(acc[0], acc[1]), add_2, o[2 * i]);
      o[2 * i + 1] = fma2(pair(acc[2], acc[3]), add_2, o[2 * i + 1]);
    }
  }
  __device__ __forceinline__ int least() const { return __reduce_min_sync(0xffffffffu, lim); }
  // result [ROWS][PITCH], (maximum, sum) [ROWS][2]
  __device__ __forceinline__ void store(float *so, float *sml, int rows, int lane) {
    const int g = lane >> 2, t = lane & 3;
    l += __shfl_xor_sync(0xffffffffu, l, 4);
    l += __shfl_xor_sync(0xffffffffu, l, 8);
    l += __shfl_xor_sync(0xffffffffu, l, 16);
    if (t >= rows) return;
    if (g == 0) sml[2 * t] = m, sml[2 * t + 1] = l;
#pragma unroll
    for (int i = 0; i < HDP / 8; i++) {
      const float2 v = unpair(o[i]);
      so[t * PITCH + 8 * i + g] = v.x + v.y;
    }
  }
};

// Five to eight (RG = 1) or nine to sixteen rows (RG = 2): the query rows are the row operand, values in the upper and residues
// in the lower 8 rows, codes its 8 columns: lane (g, t) has the scores of rows 8r + g at positions 8t .. 8t + 7.
template <int HDP, int RG>
struct ManyRows {
  static constexpr int ROWS = 8 * RG, KS = HDP / 16, NT = HDP / 8, PITCH = HDP + 8, RESIDENT = HDP * RG <= 64 ? 4 : HDP * RG <= 128 ? 3 : 2;
  uint32_t qf[RG][KS][4];
  float qs[RG], m[RG], l[RG];
  uint64_t o[RG][NT];
  int lim[RG];

  __device__ __forceinline__ void start(const AttnParams &p, int s, int h, int row0, const Sight &sight, int lane) {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int r = 0; r < RG; r++) {
      const int row = row0 + r * 8 + g;
      float x[KS][4];
      qs[r] = load_row<KS>(p, s, h, row, t, x);
#pragma unroll
      for (int k = 0; k < KS; k++) {
        split2(x[k][0], x[k][1], qf[r][k][0], qf[r][k][1]);
        split2(x[k][2], x[k][3], qf[r][k][2], qf[r][k][3]);
      }
      lim[r] = row < p.G * p.T ? sight.limit(row / p.G) : sight.len;
      m[r] = -INFINITY, l[r] = 0.0f;
#pragma unroll
      for (int i = 0; i < NT; i++) o[r][i] = 0;
    }
  }

  // `all`: every row sees every position of the block
  __device__ __forceinline__ void block(const uint8_t *sb, int first, bool all, int lane) {
    const int t = lane & 3;
    float sc[RG][4][4];
#pragma unroll
    for (int r = 0; r < RG; r++)
#pragma unroll
      for (int j = 0; j < 4; j++) sc[r][j][0] = sc[r][j][1] = sc[r][j][2] = sc[r][j][3] = 0.0f;
#pragma unroll
    for (int c = 0; c < KS; c++) {
      const uint4 w4 = *(const uint4 *)(sb + c * 512 + lane * 16);
      const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
      for (int u = 0; u < 4; u++) {
        uint32_t x, y;
        widen(w[u], x, y);
        const int j = (4 * c + u) / KS, k = (4 * c + u) % KS;
#pragma unroll
        for (int r = 0; r < RG; r++) mma(sc[r][j], qf[r][k][0], qf[r][k][1], qf[r][k][2], qf[r][k][3], x, y);
      }
    }
    const float2 scales = *(const float2 *)(sb + 2 * kBlock * HDP);
    uint32_t pf[RG][2][4];
    float add[RG];
#pragma unroll
    for (int r = 0; r < RG; r++) {
      const int n = lim[r] - first - 8 * t;  // this lane's positions 0..n-1 are seen
      const float f = scales.x * kScoreUnit * qs[r];
      float v[4][2], top = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; j++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          v[j][e] = (sc[r][j][e] + sc[r][j][2 + e]) * f;
          if (!all) v[j][e] = 2 * j + e < n ? v[j][e] : -INFINITY;
          top = fmaxf(top, v[j][e]);
        }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const float ref = top - kUpW, M = fmaxf(m[r], ref), c = rescale(ref, M), from = ref == -INFINITY ? 0.0f : ref;
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; j++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          v[j][e] = ex2(v[j][e] - from);
          sum += v[j][e];
        }
      const float old = rescale(m[r], M);
      l[r] = fmaf(l[r], old, sum * c);
      if (__any_sync(0xffffffffu, old != 1.0f)) {
        const uint64_t old_2 = pair(old, old);
#pragma unroll
        for (int i = 0; i < NT; i++) o[r][i] = mul2(o[r][i], old_2);
      }
      add[r] = lim[r] > first ? c * scales.y : 0.0f;  // (a block that a row sees nothing of may hold NaN)
      m[r] = M;
#pragma unroll
      for (int kk = 0; kk < 2; kk++) {
        split2(v[2 * kk][0], v[2 * kk][1], pf[r][kk][0], pf[r][kk][1]);
        split2(v[2 * kk + 1][0], v[2 * kk + 1][1], pf[r][kk][2], pf[r][kk][3]);
      }
    }
#pragma unroll
    for (int c = 0; c < KS; c++) {
      const uint4 w4 = *(const uint4 *)(sb + kBlock * HDP + c * 512 + lane * 16);
      const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
      for (int u = 0; u < 2; u++) {
        uint32_t x0, y0, x1, y1;
        widen(w[2 * u], x0, y0);
        widen(w[2 * u + 1], x1, y1);
#pragma unroll
        for (int r = 0; r < RG; r++) {
          float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
          mma(acc, pf[r][0][0], pf[r][0][1], pf[r][0][2], pf[r][0][3], x0, y0);
          mma(acc, pf[r][1][0], pf[r][1][1], pf[r][1][2], pf[r][1][3], x1, y1);
          uint64_t &d = o[r][2 * c + u];
          d = fma2(add2(pair(acc[0], acc[1]), pair(acc[2], acc[3])), pair(add[r], add[r]), d);
        }
      }
    }
  }
  __device__ __forceinline__ int least() const {
    int v = lim[0];
#pragma unroll
    for (int r = 1; r < RG; r++) v = min(v, lim[r]);
    return __reduce_min_sync(0xffffffffu, v);
  }
  __device__ __forceinline__ void store(float *so, float *sml, int rows, int lane) {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int r = 0; r < RG; r++) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      const int row = r * 8 + g;
      if (row >= rows) continue;
      if (t == 0) sml[2 * row] = m[r], sml[2 * row + 1] = l[r];
#pragma unroll
      for (int i = 0; i < NT; i++) *(float2 *)(so + row * PITCH + 8 * i + 2 * t) = unpair(o[r][i]);
    }
  }
};

// Blocks on their way per warp: 4 KB each at 64 channels, three thread blocks an SM, so 192 KB an SM.  (More of them, or more
// warps, gave nothing; blocks a multiple of 128 bytes apart neither.)
template <int HDP>
__host__ __device__ constexpr int stages() { return HDP <= 32 ? 8 : HDP <= 64 ? 4 : HDP <= 128 ? 2 : 1; }
// rings, then two results of each warp, `rows` rows each
template <int HDP, class Acc>
__host__ __device__ constexpr size_t smem_bytes(int rows = Acc::ROWS) {
  return (size_t)kWarps * stages<HDP>() * kv8::block_bytes(HDP) + (size_t)2 * kWarps * rows * (Acc::PITCH + 2) * 4;
}
// What a unit costs a warp beside its blocks (queries, its result), in blocks: shares of the list are equal with it.
constexpr int kTurn = 4;
constexpr int kLeast = 2;  // places of a warp's share at least
// Places of a launch at most, unless one group of rows alone has more: the kernel counts them in 32 bits, a warp's share beyond the
// end included.  Several launches of 2^24 places take milliseconds each, so that what a further one costs does not show.
constexpr long long kMostPlaces = 1 << 24;

// Result row from its parts: maximum and sum of weights, channels lane, lane + 32, ...
template <int HDP>
struct Joined {
  float M = -INFINITY, L = 0.0f, a[HDP / 32];
  __device__ __forceinline__ Joined() {
#pragma unroll
    for (int i = 0; i < HDP / 32; i++) a[i] = 0.0f;
  }
  __device__ __forceinline__ void add(float m, float l, const float (&v)[HDP / 32]) {
    const float top = fmaxf(M, m), f = rescale(M, top), w = rescale(m, top);
    M = top, L = fmaf(L, f, l * w);
#pragma unroll
    for (int i = 0; i < HDP / 32; i++) a[i] = fmaf(a[i], f, v[i] * w);
  }
  __device__ __forceinline__ void finish(const AttnParams &p, int s, int h, int row, bool sees, int lane) const {
    const int i = row / p.G, C = p.H * p.G * p.HD, col0 = (h * p.G + row - i * p.G) * p.HD;
    const long long orow = (long long)s * p.T + i;
    const float inv = 1.0f / L;
#pragma unroll
    for (int k = 0; k < HDP / 32; k++) {
      const int d = lane + 32 * k, col = col0 + d;
      if (d >= p.HD) break;
      const float y = sees ? a[k] * inv : 0.0f;
      p.out[orow * C + col] = y;
      if (p.y16) {
        __half *d16 = p.y16 + ((long long)(col >> 6) * p.R + orow) * 64 + (col & 63);
        const __half hi = __float2half_rn(y);
        *d16 = hi;
        if (p.lo_off) d16[p.lo_off] = __float2half_rn(y - __half2float(hi));
      }
    }
  }
};

// All blocks of all units (stream, head, group of rows) form one list, of which every warp takes an equal share and streams it
// through a ring of its own that the copy engine keeps full across the units' borders: no barrier, and no warp waits for
// another's blocks.  A unit inside a share is finished by its warp.  The others meet first in the thread block, whose warps'
// shares are neighbours, then, where a unit lies in several thread blocks, in the one that takes the last ticket; parts are
// joined in the list's order (nothing waits, and the result does not depend on who comes last).
//
// Bound by HBM where blocks are many: 64 streams, one token, 20 heads of 64 over 1500 positions (247 MB) 51.7 us = 4.8 TB/s; 4
// streams, 32 query heads on 8 of 128, 65551 positions (538 MB) 98 us = 5.5 TB/s; by a chain of latencies where they are few
// (one stream of the former 8.9 us).  What is left of the former is that the SMs stream at different rates, so that equal shares
// end 15 % apart.  Shares that warps claim one after the other even that out and cost more, in starts, results and joins, than
// they give (58 to 80 us by their size), as do two or three thread blocks a place on the GPU (58, 64).
template <int HDP, class Acc>
__global__ void __launch_bounds__(kThreads, Acc::RESIDENT) k_attn_kv8(const AttnParams p) {
  constexpr int BB = (int)kv8::block_bytes(HDP), NST = stages<HDP>(), ROWS = Acc::ROWS, PITCH = Acc::PITCH, NK = HDP / 32;
  extern __shared__ __align__(128) uint8_t ring[];  // [kWarps][NST][BB], then results [2*kWarps][rows][PITCH] and [2*kWarps][rows][2]
  __shared__ __align__(8) uint64_t full[kWarps][NST];
  __shared__ int found[kWarps][3];      // unit, first block and unit's place in the list at the start of a warp's share
  __shared__ int scan[kWarps];
  __shared__ int part_unit[2 * kWarps], part_base[2 * kWarps];
  __shared__ int open_unit[2], open_base[2], last[2];  // units that lie in other thread blocks too: before this one, behind it
  const int nrows = p.G * p.T, rows = min(ROWS, nrows);
  float *res = (float *)(ring + kWarps * NST * BB), *resml = res + 2 * kWarps * rows * PITCH;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x < kWarps * NST) tc::mbar_init(smem_u32(&full[0][0] + threadIdx.x), 1);
  if (threadIdx.x < 2 * kWarps) part_unit[threadIdx.x] = -1;
  if (threadIdx.x < 2) open_unit[threadIdx.x] = -1;
  tc::fence_barrier_init();
  __syncthreads();
  Sight sight;
  bool bad;
  const int each = p.H * p.rowgroups;  // units of a stream
  const bool ragged = p.lens || p.rows.pos || p.rows.counts;
  // Where the launch in front is the one that writes this call's rows (which lets go of this one only when all before it has
  // ended), the first blocks that it does not touch are fetched while it runs.
  const int ready = p.causal && !ragged ? p.rows.n / kBlock : 0;
  if (ready) fa_grid_dep_launch();
  else fa_grid_dep_sync();
  const int shares = (int)gridDim.x * kWarps, mine = (int)blockIdx.x * kWarps + warp;
  int total = 0, per, unit = 0, b0 = 0, base = 0;  // places, a share, its first unit, first block in that, the unit's place in the list
  if (!ragged) {
    sight.of(p, 0, bad);
    const int nb = sight.blocks() + kTurn;
    total = p.S * each * nb;
    per = (total + shares - 1) / shares;
    const int f0 = min(mine * per, total);
    unit = f0 / nb, b0 = f0 - unit * nb, base = unit * nb;
  } else {  // streams of different lengths: each thread sums a run of them, the one that holds a share's start looks closer
    const int run = (p.S + kThreads - 1) / kThreads, s0 = min((int)threadIdx.x * run, p.S), s1 = min(s0 + run, p.S);
    int sum = 0;
    for (int s = s0; s < s1; s++) {
      sight.of(p, s, bad);
      if (bad && blockIdx.x == 0) atomicOr(p.status + 3, kStatusKv8Length);
      sum += (sight.blocks() + kTurn) * each;
    }
    int upto = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    if (lane == 31) scan[warp] = upto;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; w++) {
      if (w < warp) upto += scan[w];
      total += scan[w];
    }
    per = (total + shares - 1) / shares;
#pragma unroll
    for (int w = 0; w < kWarps; w++) {
      const int f0 = ((int)blockIdx.x * kWarps + w) * per;
      if (f0 < upto - sum || f0 >= upto) continue;
      int at = upto - sum, s = s0;
      for (;; s++) {
        sight.of(p, s, bad);
        if (f0 < at + (sight.blocks() + kTurn) * each) break;
        at += (sight.blocks() + kTurn) * each;
      }
      const int nb = sight.blocks() + kTurn, h = (f0 - at) / nb;
      found[w][0] = s * each + h, found[w][1] = f0 - at - h * nb, found[w][2] = at + h * nb;
    }
    __syncthreads();
    if (mine * per < total) unit = found[warp][0], b0 = found[warp][1], base = found[warp][2];
  }
  if ((int)blockIdx.x * kWarps * per >= total) return;  // (the whole thread block)
  const int f1 = min((mine + 1) * per, total);
  auto place = [&](int u, int &s, int &h, int &row0) {
    const int sh = u / p.rowgroups;
    s = sh / p.H, h = sh - s * p.H, row0 = (p.rg0 + u - sh * p.rowgroups) * ROWS;
  };
  int s, h, row0;
  bool ok = true;
  if (mine * per < total) {
    place(unit, s, h, row0);
    sight.of(p, s, bad);
    if (b0 >= sight.blocks()) base += sight.blocks() + kTurn, unit++, b0 = 0;  // the share begins behind a unit's blocks
  } else {
    base = f1;
  }
  if (base >= f1) {
    if (ready) fa_grid_dep_wait();
  } else {
    place(unit, s, h, row0);
    sight.of(p, s, bad);
    const uint32_t slots = smem_u32(ring) + warp * (NST * BB), bars = smem_u32(&full[warp][0]);
    // the next block to fetch
    int pu = unit, pbase = base, pnb = sight.blocks(), pleft = min(pnb, f1 - pbase) - b0, pst = 0;
    const uint8_t *psrc = p.codes + ((size_t)(pu / p.rowgroups) * p.nblk + b0) * BB;
    int pb = b0;  // (kept for the first fetches)
    bool waited = ready == 0;
    auto fetch = [&](bool first) {  // (all lanes keep the place, one issues)
      if (pleft == 0) {
        pbase += pnb + kTurn, pu++;
        if (pbase >= f1) {
          pbase -= pnb + kTurn, pu--;
          return;
        }
        if (ragged) {
          Sight next;
          bool b;
          next.of(p, pu / each, b);
          pnb = next.blocks();
        }
        pleft = min(pnb, f1 - pbase);
        psrc = p.codes + (size_t)(pu / p.rowgroups) * p.nblk * BB;
        pb = 0;
      }
      if (first && !waited && pb++ >= ready) fa_grid_dep_wait(), waited = true;
      if (lane == 0) {
        tc::mbar_expect_tx(bars + 8 * pst, BB);
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(slots + pst * BB),
                     "l"(psrc), "r"(BB), "r"(bars + 8 * pst)
                     : "memory");
      }
      psrc += BB, pleft--;
      if (++pst == NST) pst = 0;
    };
#pragma unroll 1
    for (int k = 0; k < NST; k++) fetch(true);
    if (!waited) fa_grid_dep_wait();

    int st = 0, parity = 0;
#pragma unroll 1
    for (;;) {  // one unit, or the part of it in this share
      const int nb = sight.blocks(), b1 = min(nb, f1 - base);
      Acc acc;
      acc.start(p, s, h, row0, sight, lane);
      const int least = acc.least();
#pragma unroll 1
      for (int b = b0; b < b1; b++) {
        ok = __all_sync(0xffffffffu, tc::mbar_wait(bars + 8 * st, parity, p.wait_limit)) && ok;
        acc.block(ring + (warp * NST + st) * BB, b * kBlock, (b + 1) * kBlock <= least, lane);
        __syncwarp();
        fetch(false);
        if (++st == NST) st = 0, parity ^= 1;
      }
      const int slot = 2 * warp + (b0 == 0);  // the part in front of all others, or behind
      float *ro = res + slot * rows * PITCH, *rm = resml + slot * rows * 2;
      __syncwarp();
      acc.store(ro, rm, rows, lane);
      __syncwarp();
      if (b0 == 0 && b1 == nb) {
        for (int row = 0; row < min(rows, nrows - row0); row++) {
          Joined<HDP> j;
          float v[NK];
#pragma unroll
          for (int i = 0; i < NK; i++) v[i] = ro[row * PITCH + lane + 32 * i];
          j.add(rm[2 * row], rm[2 * row + 1], v);
          j.finish(p, s, h, row0 + row, sight.limit((row0 + row) / p.G) > 0, lane);
        }
      } else if (lane == 0) {
        part_unit[slot] = unit, part_base[slot] = base;
      }
      base += nb + kTurn, unit++, b0 = 0;
      if (base >= f1) break;
      place(unit, s, h, row0);
      sight.of(p, s, bad);
    }
    if (!ok && lane == 0) {
      atomicExch(p.status, 81);
      p.status[1] = blockIdx.x, p.status[2] = warp;
    }
  }
  __syncthreads();

  // parts of the thread block's warps; a unit's parts are neighbours
  const int share = kWarps * per, first = (int)blockIdx.x * share;
  for (int i = 0, group = 0; i < 2 * kWarps;) {
    const int u = part_unit[i];
    if (u < 0) {
      i++;
      continue;
    }
    int end = i + 1;
    while (end < 2 * kWarps && (part_unit[end] < 0 || part_unit[end] == u)) end++;
    if ((group++ & (kWarps - 1)) == warp) {
      const int at = part_base[i];
      place(u, s, h, row0);
      sight.of(p, s, bad);
      const bool whole = at >= first && at + sight.blocks() <= first + share;
      const int side = at >= first;
      for (int row = 0; row < min(rows, nrows - row0); row++) {
        Joined<HDP> j;
        for (int k = i; k < end; k++) {
          if (part_unit[k] < 0) continue;
          float v[NK];
#pragma unroll
          for (int c = 0; c < NK; c++) v[c] = res[(k * rows + row) * PITCH + lane + 32 * c];
          j.add(resml[(k * rows + row) * 2], resml[(k * rows + row) * 2 + 1], v);
        }
        if (whole) {
          j.finish(p, s, h, row0 + row, sight.limit((row0 + row) / p.G) > 0, lane);
        } else {
          const size_t part = ((size_t)blockIdx.x * 2 + side) * rows + row;
#pragma unroll
          for (int c = 0; c < NK; c++) p.pacc[part * HDP + lane + 32 * c] = j.a[c];
          if (lane == 0) *(float2 *)(p.pml + part * 2) = make_float2(j.M, j.L);
        }
      }
      if (!whole && lane == 0) open_unit[side] = u, open_base[side] = at;
    }
    i = end;
  }
  __threadfence();
  __syncthreads();
  if (open_unit[0] < 0 && open_unit[1] < 0) return;
  if (threadIdx.x < 2) {
    const int u = open_unit[threadIdx.x];
    last[threadIdx.x] = 0;
    if (u >= 0) {
      place(u, s, h, row0);
      sight.of(p, s, bad);
      const int at = open_base[threadIdx.x], others = (at + sight.blocks() - 1) / share - at / share;
      last[threadIdx.x] = atomicAdd(p.tickets + u, 1) == others;
      if (last[threadIdx.x]) p.tickets[u] = 0;  // ready for the next launch on this stream
    }
  }
  __syncthreads();
  for (int k = 0; k < 2; k++) {
    if (!last[k]) continue;
    __threadfence();
    const int at = open_base[k];
    place(open_unit[k], s, h, row0);
    sight.of(p, s, bad);
    const int c0 = at / share, c1 = (at + sight.blocks() - 1) / share;
    for (int row = warp; row < min(rows, nrows - row0); row += kWarps) {
      Joined<HDP> j;
      constexpr int kParts = HDP <= 64 ? 8 : 4;  // in flight together
      for (int c = c0; c <= c1; c += kParts) {
        float2 ml[kParts];
        float v[kParts][NK];
#pragma unroll
        for (int n = 0; n < kParts; n++) {
          const int cc = min(c + n, c1);
          const size_t part = ((size_t)cc * 2 + (at >= cc * share)) * rows + row;
          ml[n] = __ldcg((const float2 *)(p.pml + part * 2));
#pragma unroll
          for (int i = 0; i < NK; i++) v[n][i] = __ldcg(p.pacc + part * HDP + lane + 32 * i);
        }
#pragma unroll
        for (int n = 0; n < kParts; n++)
          if (c + n <= c1) j.add(ml[n].x, ml[n].y, v[n]);
      }
      j.finish(p, s, h, row0 + row, sight.limit((row0 + row) / p.G) > 0, lane);
    }
  }
}

// Resident thread blocks per SM of a kernel, asked once.
template <int HDP, class Acc>
int resident(int rows) {
  static std::atomic<int> asked[Acc::ROWS];
  auto &known = asked[rows - 1];
  int n = known.load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, k_attn_kv8<HDP, Acc>, kThreads, smem_bytes<HDP, Acc>(rows)) != cudaSuccess || n < 1) n = 1;
    known.store(n, std::memory_order_relaxed);
  }
  return n;
}

template <int HDP, class Acc>
int run(fa_ctx *ctx, const fa_kv8 *c, AttnParams &p, int most, const char *label) {
  constexpr int ROWS = Acc::ROWS;
  static SmemLimit limit;
  FA_CHECK_CUDA(ctx, limit.raise(ctx, k_attn_kv8<HDP, Acc>, smem_bytes<HDP, Acc>()));
  const int nb = ceil_div(most < 1 ? 1 : most, kBlock), groups = ceil_div(p.G * p.T, ROWS);
  const long long list = (long long)c->S * c->H * (nb + kTurn);  // places of a row group, < 2^29: the cache fits the device
  const int rows = p.G * p.T < ROWS ? p.G * p.T : ROWS, slots = ctx->sm_count * resident<HDP, Acc>(rows);
  int rc = FA_OK;
  for (p.rg0 = 0; p.rg0 < groups && rc == FA_OK; p.rg0 += p.rowgroups) {
    const long long fit = list < kMostPlaces ? kMostPlaces / list : 1;
    p.rowgroups = (int)(groups - p.rg0 < fit ? groups - p.rg0 : fit);
    const long long share = (list * p.rowgroups + kWarps * kLeast - 1) / (kWarps * kLeast);
    const int grid = (int)(share < slots ? share : slots);
    // room for all thread blocks that the GPU holds, whatever the grid: a cache that grows block by block wants the same memory
    const size_t part = (size_t)slots * 2 * rows, tickets = p.rowgroups > 1 ? (size_t)c->S * c->H * p.rowgroups : 0;
    void *scratch = nullptr;
    size_t bytes = 0;
    FA_TRY(fa_block_acquire(ctx, part * (HDP + 2) * 4 + tickets * 4, &scratch, &bytes));
    p.pacc = (float *)scratch, p.pml = p.pacc + part * HDP;
    p.tickets = c->tickets;
    cudaError_t e = cudaSuccess;
    if (tickets) {
      p.tickets = (int *)(p.pml + part * 2);
      e = cudaMemsetAsync(p.tickets, 0, tickets * 4, ctx->stream);
    }
    if (e == cudaSuccess) {
      LaunchScope ls(ctx, label);
      e = fa_launch_dep(ctx, k_attn_kv8<HDP, Acc>, dim3(grid), dim3(kThreads), smem_bytes<HDP, Acc>(rows), p);
    }
    if (e != cudaSuccess) rc = fa_fail(ctx, FA_ERR_CUDA, "launch %s: %s", label, cudaGetErrorString(e));
    fa_block_release(ctx, scratch);
  }
  return rc;
}

// ---- many rows: prompts, or many query heads to a key head ---------------------------------------------------------------
//
// 128 rows of a unit against 128 positions at a time on tcgen05: S = Q K^T and O = P V with the accumulators in TMEM, a row to
// a lane.  Eight warps, two threads a row with half of the positions each, turn cache blocks into the f16 tiles of K (position
// by channel) and V^T (channel by position) in the swizzled K-major layout that the tensor cores read, and do the softmax; a
// ninth issues the products.  Both products run twice, with the value and the residue of the rows' side.  P takes the place of
// S in TMEM, 32 positions at a time (16 columns of values, 16 of residues), and is the TMEM operand of the second product.
// The next tile's K is made while a tile's P V runs and its V while its own scores are computed.
//
// A row of P holds the weights times their blocks' value scales, relative to the largest such product that this row has in this
// tile and times 2^kUpP, so that the whole f16 range is for what counts to the row, and the accumulator needs no scale per block.
// What other rows see, or blocks that a row gives no weight to, however large their values, is not in it.  A tile's result
// joins the running one, which has a reference of its own and lies in TMEM beside it.  The sum of the weights alone is kept
// relative to the largest score; it takes the scales out of the sums of products again, a factor for each block.  References are whole
// powers of two: what moves between them is not rounded, up to scores of 2^23.  (Weights formed relative to their own block's largest
// and multiplied with its scale afterwards would take scores of any size and no logarithm of a scale: 64 us in place of 57, the same
// error.)
//
// What bounds it: the chain of a tile's scores, softmax and products, which two thread blocks an SM overlap where shared memory
// allows, and a thread block's start and end, a few tiles' worth.  8 streams of 224 queries, 20 heads of 64 over up to 1500
// positions of different lengths: 57 us, in which 2.1 of 4 instructions a clock are issued (23 a score, all in all) and the tensor
// pipe is busy for 22 %; 16 streams' prompts of 224 over themselves: write and attention 54 us.
// Separate warps for the softmax and the conversion took 70 us in place of 55, runs of four to eight tiles 72 to 80.
// From this many rows of a unit on.  Measured, us, groups of 16 rows / this kernel, 16 streams of 20 heads of 64 over 1500
// positions: 32 rows 62 / 95, 48 rows 81 / 99, 64 rows 96 / 95; one stream: 24 rows 25 / 20, 64 rows 27 / 19.  The rule goes by
// the former, whose loss is the larger one; other widths and lengths were not measured for it.
constexpr int kPromptRows = 49;
constexpr int kTile = 128, kPromptThreads = 288, kUpP = 6;
// A block's scale is taken for so large at least that a weight at the row's maximum gives 2^-kFar of the largest product (0, as
// f16): products as small as f32 may have them would take the weights out of their sum.
constexpr float kFar = 80.0f;

template <int HDP>
struct PromptSmem {
  static constexpr int CH = (HDP + 63) / 64;                                      // 64-channel chunks of a row
  static constexpr int Q = 0, K = Q + 2 * CH * 16384, V = K + CH * 16384, STAGE = V + 2 * HDP * 128;
  static constexpr int STAGE_BYTES = (4 * (int)kv8::block_bytes(HDP) + 127) / 128 * 128, BYTES = STAGE + 2 * STAGE_BYTES + 1024;
};

__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, "
      "%20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]),
      "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]),
      "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]),
      "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// 32 columns of this thread's lane
__device__ __forceinline__ void tmem_ld32(uint32_t addr, float (&v)[32]) {
  uint32_t a[16], b[16];
  tc::tmem_ld16(addr, a);
  tc::tmem_ld16(addr + 16, b);
  tc::tmem_ld_wait();
#pragma unroll
  for (int i = 0; i < 16; i++) v[i] = __uint_as_float(a[i]), v[16 + i] = __uint_as_float(b[i]);
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// D (+)= A B with A in TMEM (16 f16 of a row in 8 columns) and B in shared memory
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

struct PromptParams {
  AttnParams a;
  int rowtiles, splits, per;  // row tiles of a unit, splits of the positions and their tiles
};

template <int HDP>
__global__ void __launch_bounds__(kPromptThreads, HDP <= 64 ? 2 : 1) k_prompt_kv8(const PromptParams pp) {
  using Smem = PromptSmem<HDP>;
  constexpr int KS = HDP / 16, CH = Smem::CH, BB = (int)kv8::block_bytes(HDP), kWaits = 81, kColumns = HDP <= 64 ? 256 : 512;
  const AttnParams &p = pp.a;
  extern __shared__ uint8_t raw_smem[];
  uint8_t *smem = raw_smem + ((1024 - (smem_u32(raw_smem) & 1023)) & 1023);
  __shared__ __align__(8) uint64_t bar[9];  // see the names below
  __shared__ float tops[2][2][kTile];        // row maxima of the two halves; their sums of weights and maxima in the end
  __shared__ float scl[2][4][4];            // a tile's scales: keys, in units of log 2; values as 2^[1] * 2^[2], and 2^-[2]
  __shared__ uint32_t tmem_slot;
  __shared__ int gave_up;
  const uint32_t s_full = smem_u32(&bar[0]), p_full = smem_u32(&bar[1]), pv_done = smem_u32(&bar[2]), k_full = smem_u32(&bar[3]),
                 v_full = smem_u32(&bar[4]), code_free = smem_u32(&bar[5]), code_full = smem_u32(&bar[6]),  // (two stages)
                 drained = smem_u32(&bar[8]);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  int at = blockIdx.x;
  const int split = at % pp.splits;
  at /= pp.splits;
  const int rt = pp.rowtiles - 1 - at % pp.rowtiles, unit = at / pp.rowtiles, s = unit / p.H, h = unit - s * p.H;  // (longest first)
  if (tid == 0) {
    tc::mbar_init(s_full, 2);  // the products, and who issued them: the scales of the tile come with it
    tc::mbar_init(p_full, 8);  // one arrival a warp here and below: a lane's own would come one after the other
    tc::mbar_init(pv_done, 1);
    tc::mbar_init(k_full, 8);
    tc::mbar_init(v_full, 8);
    tc::mbar_init(code_free, 8);
    tc::mbar_init(code_full, 1);
    tc::mbar_init(code_full + 8, 1);
    tc::mbar_init(drained, 1);
    tc::fence_barrier_init();
    gave_up = 0;
  }
  if (warp == 8) tc::tmem_alloc(smem_u32(&tmem_slot), kColumns);
  __syncthreads();  // in front of the next grid's start, which may want columns too
  fa_grid_dep_sync();

  Sight sight;
  bool bad;
  sight.of(p, s, bad);
  if (bad && tid == 0) atomicOr(p.status + 3, kStatusKv8Length);
  const int nrows = p.G * p.T, row_a = rt * kTile, row_b = min(nrows, row_a + kTile) - 1;
  int most = sight.len;
  if (p.causal) {
    const int i = min(row_b / p.G, sight.count - 1);
    most = i >= row_a / p.G ? sight.start + i + 1 : 0;
  }
  const int t0 = split * pp.per, t1 = min((most + kTile - 1) / kTile, t0 + pp.per), nt = max(0, t1 - t0);
  const uint8_t *codes = p.codes + (size_t)unit * p.nblk * BB;

  // everything that is read first is asked for together: the codes of two tiles, the query rows
  auto fetch = [&](int k) {  // tile k of this range into stage k & 1
    const int b = (t0 + k) * 4, n = min(4, p.nblk - b);
    const uint32_t bytes = (uint32_t)n * BB, dst = smem_u32(smem + Smem::STAGE + (k & 1) * Smem::STAGE_BYTES), on = code_full + 8 * (k & 1);
    tc::mbar_expect_tx(on, bytes);
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(codes + (size_t)b * BB),
                 "r"(bytes), "r"(on)
                 : "memory");
  };
  int fetched = min(2, nt);  // tiles asked for
  if (tid == 0)
    for (int k = 0; k < fetched; k++) fetch(k);
  // a row's channels over LPR lanes
  constexpr int LPR = HDP <= 32 ? 8 : HDP <= 64 ? 16 : 32, PER = LPR / 2;  // rows of a thread
  const int sub = tid & (LPR - 1), d0 = sub * 4, line = tid / LPR;
  auto of_row = [&](int r, int &i, int &head) {  // row of the tile -> query, query head
    const int rr = min(row_a + r, nrows - 1);
    i = rr / p.G, head = h * p.G + rr - i * p.G;
  };
  float4 x[PER];
  if (warp < 8) {
#pragma unroll
    for (int k = 0; k < PER; k++) {
      const int r = line + k * (256 / LPR);
      int i, head;
      of_row(r, i, head);
      const float *qp = p.q + ((long long)s * p.T + i) * p.ldq + head * p.HD + d0;
      x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (row_a + r < nrows && d0 < p.HD) {
        if (p.vec) {
          x[k] = *(const float4 *)qp;
        } else {
          x[k].x = qp[0];
          if (d0 + 1 < p.HD) x[k].y = qp[1];
          if (d0 + 2 < p.HD) x[k].z = qp[2];
          if (d0 + 3 < p.HD) x[k].w = qp[3];
        }
      }
    }
  }
  // queries scaled and split as in load_row
  if (warp < 8) {
#pragma unroll
    for (int k = 0; k < PER; k++) {
      const int r = line + k * (256 / LPR);
      uint32_t a = max(max(__float_as_uint(x[k].x) & 0x7fffffffu, __float_as_uint(x[k].y) & 0x7fffffffu),
                       max(__float_as_uint(x[k].z) & 0x7fffffffu, __float_as_uint(x[k].w) & 0x7fffffffu));
#pragma unroll
      for (int o = 1; o < LPR; o <<= 1) a = max(a, __shfl_xor_sync(0xffffffffu, a, o));
      const int bits = (int)(a >> 23), ex = min(max(bits, kUp + 1), 254);
      const float f = __int_as_float((254 + kUp - ex) << 23);
      if (sub == 0) tops[0][0][r] = bits < 255 ? __int_as_float(ex << 23) : __int_as_float(0x7fc00000);
      if (d0 < HDP) {
        uint2 hi, lo;
        split2(x[k].x * f, x[k].y * f, hi.x, lo.x);
        split2(x[k].z * f, x[k].w * f, hi.y, lo.y);
        uint8_t *dst = smem + Smem::Q + (d0 >> 6) * 16384 + r * 128 + ((((d0 & 63) >> 3) ^ (r & 7)) << 4) + (d0 & 4) * 2;
        *(uint2 *)dst = hi;
        *(uint2 *)(dst + CH * 16384) = lo;
      }
    }
    tc::fence_proxy_async_smem();
  }
  const int quad = warp & 3, half = warp >> 2, local = quad * 32 + lane, row = row_a + local;
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = tmem_slot, tS = tmem, tO = tmem + 128, tSum = tO + HDP;
  const float qs = tops[0][0][local];
  __syncthreads();  // (the array's next use)
  // Where a wait runs out a thread goes on without waiting for anything: every loop ends, every barrier gets its arrivals, and
  // the status word makes the result void.
  bool ok = true;
  auto wait = [&](uint32_t b, uint32_t parity) {
    if (ok) ok = tc::mbar_wait(b, parity, p.wait_limit);
  };
  // this thread's half of the row: reference and sum of its weights; both halves: references of the running result, of a tile's
  float m = -INFINITY, l = 0.0f, run_ref = -INFINITY, tile_ref = -INFINITY;

  if (warp < 8) {
    const int g = lane >> 2, t = lane & 3;
    auto arrive = [&](uint32_t b) {
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(b);
    };
    // a warp's share of tile k: block `quad`, half of its channels
    auto stage = [&](int k) { return smem + Smem::STAGE + (k & 1) * Smem::STAGE_BYTES + quad * BB; };
    auto keys = [&](int k) {
      wait(code_full + 8 * (k & 1), (k >> 1) & 1);
      __syncwarp();
      const uint8_t *blk = stage(k);
      // position r = 32 quad + 8 (g/2) + 2j + g%2, 16-byte unit 2 (ks%4) + t/2 of its row: swizzled, 2 (ks%4 ^ j) + (t/2 ^ g%2)
      uint8_t *dst = smem + Smem::K + (quad * 32 + 8 * (g >> 1) + (g & 1)) * 128 + (((t >> 1) ^ (g & 1)) << 4) + (t & 1) * 8;
      auto part = [&](auto which) {
        constexpr int kHalf = decltype(which)::value;
#pragma unroll
        for (int c = kHalf * (KS / 2); c < (kHalf + 1) * (KS / 2); c++) {
          const uint4 w4 = *(const uint4 *)(blk + c * 512 + lane * 16);
          const uint32_t word[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
          for (int u = 0; u < 4; u++) {
            const int j = (4 * c + u) / KS, ks = (4 * c + u) % KS;
            uint2 x;
            widen(word[u], x.x, x.y);
            *(uint2 *)(dst + (ks >> 2) * 16384 + j * 256 + (((ks & 3) ^ j) << 5)) = x;
          }
        }
      };
      if (half == 0) part(std::integral_constant<int, 0>());
      else part(std::integral_constant<int, 1>());
      if (half == 0 && lane == 0) {
        const bool there = (t0 + k) * 4 + quad < p.nblk;
        const float2 sc = there ? *(const float2 *)(blk + 2 * kBlock * HDP) : make_float2(0.f, 0.f);
        // sc.y = 2^e * f, f in [1, 2).  A scale of 0 stands with codes of 0, so it may be any: 2^-200 is below all others.
        const bool small = sc.y < 1e-30f;
        const uint32_t bits = __float_as_uint(small ? sc.y * 0x1p64f : sc.y);
        const float f = sc.y < INFINITY ? __uint_as_float((bits & 0x7fffffu) | 0x3f800000u) : __int_as_float(0x7fc00000);
        scl[k & 1][quad][0] = sc.x * kScoreUnit;
        scl[k & 1][quad][1] = sc.y > 0.0f ? (float)((int)(bits >> 23) - (small ? 191 : 127)) : -200.0f;
        const float lf = __log2f(f);
        scl[k & 1][quad][2] = lf, scl[k & 1][quad][3] = ex2(-lf);
      }
      tc::fence_proxy_async_smem();
      arrive(k_full);
    };
    auto values = [&](int k) {
      const uint8_t *blk = stage(k) + kBlock * HDP;
#pragma unroll
      for (int cc = 0; cc < KS / 2; cc++) {
        const int c = half * (KS / 2) + cc;
        const uint4 w4 = *(const uint4 *)(blk + c * 512 + lane * 16);
        uint4 x, y;
        widen(w4.x, x.x, x.y);
        widen(w4.y, x.z, x.w);
        widen(w4.z, y.x, y.y);
        widen(w4.w, y.z, y.w);
        const int ch = 16 * c + g, u = 4 * (quad & 1) + t;  // channels ch and ch + 8, positions 32 quad + 8t ..+7
        uint8_t *dst = smem + Smem::V + (quad >> 1) * (HDP * 128) + ch * 128 + ((u ^ (ch & 7)) << 4);
        *(uint4 *)dst = x, *(uint4 *)(dst + 1024) = y;
      }
      tc::fence_proxy_async_smem();
      arrive(v_full);
      if (lane == 0) tc::mbar_arrive(code_free);
      if (fetched < nt) {
        if (tid == 0) wait(code_free, k & 1), fetch(fetched);
        fetched++;
      }
    };
    const int lim = row < nrows ? sight.limit(row / p.G) : 0;
    const uint32_t mine = (uint32_t)(quad * 32) << 16;
    // what the tile before gave joins the running result at the larger of the two references: the tensor cores cut off what an
    // f32 cannot hold, so a sum that ran on over many tiles would shrink; within a tile the residues go first
    auto sum_up = [&](bool more) {
      const float next = fmaxf(run_ref, tile_ref), f = rescale(tile_ref, next), old = rescale(run_ref, next);
      const uint64_t f2 = pair(f, f), old2 = pair(old, old);
      run_ref = next;
#pragma unroll 1
      for (int c = half * (HDP / 2); c < (half + 1) * (HDP / 2); c += 16) {
        uint32_t x[16], y[16];
        tc::tmem_ld16(tO + mine + c, x);
        if (more) tc::tmem_ld16(tSum + mine + c, y);
        tc::tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          uint64_t v = mul2(pair(__uint_as_float(x[e]), __uint_as_float(x[e + 1])), f2);
          if (more) v = fma2(pair(__uint_as_float(y[e]), __uint_as_float(y[e + 1])), old2, v);
          const float2 r = unpair(v);
          x[e] = __float_as_uint(r.x), x[e + 1] = __float_as_uint(r.y);
        }
        tmem_st16(tSum + mine + c, x);
      }
    };
    if (nt > 0) keys(0), values(0);
    for (int k = 0; k < nt; k++) {
      wait(s_full, k & 1);
      __syncwarp();
      tc::tc_fence_after();
      const int seen = lim - (t0 + k) * kTile - 64 * half;  // of this thread's 64 positions
      float top = -INFINITY, most_of = -INFINITY;  // the largest score, the largest product of a weight and a scale
#pragma unroll 1
      for (int c = 0; c < 2; c++) {
        float v[32];
        tmem_ld32(tS + mine + 64 * half + 32 * c, v);
        const int n = seen - 32 * c;
        float t = -INFINITY;
        if (__all_sync(0xffffffffu, n >= 32)) {
#pragma unroll
          for (int e = 0; e < 32; e += 4) t = max3(t, fmaxf(v[e], v[e + 1]), fmaxf(v[e + 2], v[e + 3]));
        } else {
#pragma unroll
          for (int e = 0; e < 32; e++) t = e < n ? fmaxf(t, v[e]) : t;
        }
        const float *sc = scl[k & 1][2 * half + c];
        if (n > 0) t *= sc[0] * qs, top = fmaxf(top, t), most_of = fmaxf(most_of, t + sc[1]);  // (a NaN is no maximum)
      }
      // the product's largest for the whole row: the other half's too
      tops[k & 1][half][local] = most_of;
      asm volatile("bar.sync %0, 64;" ::"r"(1 + quad) : "memory");
      most_of = floorf(fmaxf(most_of, tops[k & 1][1 - half][local]));
      if (k > 0) sum_up(k > 1);
      tile_ref = most_of;
      const float ref = tile_ref == -INFINITY ? 0.0f : tile_ref, next = fmaxf(m, floorf(top));
      l *= rescale(m, next);
      m = next;
      const float m_or_0 = m == -INFINITY ? 0.0f : m, least_of = ref - kFar - m_or_0;
#pragma unroll 1
      for (int c = 0; c < 2; c++) {
        float v[32];
        uint32_t out[32];
        const uint32_t at = tS + mine + 64 * half + 32 * c;
        tmem_ld32(at, v);
        const int n = seen - 32 * c;
        const float *sc = scl[k & 1][2 * half + c];
        const float f = sc[0] * qs;
        // weights with the values' scale in the exponent; their sum without it
        const float whole = fmaxf(sc[1], least_of) + (kUpP - ref);
        const float shift = whole + sc[2], inv = sc[3] * ex2(-whole - m_or_0);
        const uint64_t f2 = pair(f, f), shift2 = pair(shift, shift), minus = pair(-1.0f, -1.0f);
        uint64_t sum = 0;
        auto put = [&](int e, uint64_t w) {
          sum = add2(sum, w);
          const float2 x = unpair(w);
          const __half2 hi = __floats2half2_rn(x.x, x.y);
          const float2 back = __half22float2(hi), r = unpair(fma2(pair(back.x, back.y), minus, w));
          out[e >> 1] = *(const uint32_t *)&hi, out[16 + (e >> 1)] = h2(r.x, r.y);
        };
        if (__all_sync(0xffffffffu, n >= 32)) {
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float2 z = unpair(fma2(pair(v[e], v[e + 1]), f2, shift2));
            put(e, pair(ex2(z.x), ex2(z.y)));
          }
        } else {
#pragma unroll
          for (int e = 0; e < 32; e += 2)
            put(e, pair(e < n ? ex2(fmaf(v[e], f, shift)) : 0.0f, e + 1 < n ? ex2(fmaf(v[e + 1], f, shift)) : 0.0f));
        }
        const float2 both = unpair(sum);
        if (n > 0) l = fmaf(both.x + both.y, inv, l);  // (what is not seen may have a scale that is none)
        tmem_st32(at, out);
      }
      tmem_st_wait();
      tc::tc_fence_before();
      arrive(p_full);
      if (k + 1 < nt) {  // the next tile, while the products run: K is free since the scores came, V when this tile's have run
        keys(k + 1);
        wait(pv_done, k & 1);
        __syncwarp();
        values(k + 1);
      }
    }
    if (nt > 0) wait(pv_done, (nt - 1) & 1);
    if (!ok) {
      gave_up = 1;
      if (tid == 0)  // one's own copies that may still be under way
        for (int k = max(0, nt - 2); k < nt; k++) tc::mbar_wait(code_full + 8 * (k & 1), (k >> 1) & 1, p.wait_limit);
    }
    tops[0][half][local] = l, tops[1][half][local] = m;
  }
  if (warp == 8 && lane == 0) {  // ---- products
    const uint32_t id_s = tc::make_idesc(0, kTile, kTile), id_o = tc::make_idesc(0, kTile, HDP);
    const uint64_t q0 = tc::smem_desc_sw128(smem_u32(smem + Smem::Q)), k0 = tc::smem_desc_sw128(smem_u32(smem + Smem::K)),
                   v0 = tc::smem_desc_sw128(smem_u32(smem + Smem::V));  // addresses count 16 bytes, and do not carry out of their field
    for (int k = 0; k < nt; k++) {
      wait(k_full, k & 1);
      if (k > 0) wait(pv_done, (k - 1) & 1);
      tc::tc_fence_after();
#pragma unroll
      for (int part = 0; part < 2; part++)
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
          const uint32_t off = ((ks >> 2) * 16384 + (ks & 3) * 32) / 16;
          tc::umma<0>(tS, q0 + ((1 - part) * (CH * 16384 / 16) + off), k0 + off, id_s, part + ks > 0);
        }
      tc::umma_commit(s_full);
      tc::mbar_arrive(s_full);
      wait(v_full, k & 1);
      wait(p_full, k & 1);
      tc::tc_fence_after();
#pragma unroll
      for (int part = 0; part < 2; part++)
#pragma unroll
        for (int step = 0; step < 8; step++)  // 16 positions
          umma_ts(tO, tS + (step >> 1) * 32 + (1 - part) * 16 + (step & 1) * 8, v0 + ((step >> 2) * (HDP * 128) + (step & 3) * 32) / 16, id_o,
                  part + step > 0);
      tc::umma_commit(pv_done);
    }
    if (!ok) {  // products may still be under way: they read shared memory and write columns that are given back
      gave_up = 1;
      tc::umma_commit(drained);
      tc::mbar_wait(drained, 0, p.wait_limit);
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  // the result, through shared memory (the queries' and keys' place) so that rows are written as rows
  constexpr int PITCH = HDP + 4;
  float *so = (float *)smem;
  if (warp < 8) {
    const uint32_t mine = (uint32_t)(quad * 32) << 16;
    const bool sees = row < nrows && sight.limit(row / p.G) > 0;
    const float m0 = tops[1][0][local], m1 = tops[1][1][local], M = fmaxf(m0, m1);
    const float total = tops[0][0][local] * rescale(m0, M) + tops[0][1][local] * rescale(m1, M);
    if (pp.splits > 1 && row < nrows && half == 0)
      *(float2 *)(p.pml + (((size_t)unit * pp.splits + split) * nrows + row) * 2) = make_float2(M, total);
    // from the references of the sums to the weights': 2^(end - M), in two steps, which an f32 has room for
    const float end = fmaxf(run_ref, tile_ref), tile = rescale(tile_ref, end), old = rescale(run_ref, end), away = fminf(fmaxf(end - M, -250.0f), 250.0f);
    const float part1 = floorf(away * 0.5f), part2 = ex2(away - part1);
    const float inv = (pp.splits == 1 ? 1.0f / total : 1.0f) * (1.0f / (1 << kUpP)), up = ex2(part1);
#pragma unroll 1
    for (int c = half * (HDP / 2); c < (half + 1) * (HDP / 2); c += 16) {
      uint32_t v[16];
      if (nt > 0) {
        uint32_t y[16];
        tc::tmem_ld16(tO + mine + c, v);
        if (nt > 1) tc::tmem_ld16(tSum + mine + c, y);
        tc::tmem_ld_wait();
        if (nt > 1) {
#pragma unroll
          for (int e = 0; e < 16; e++) v[e] = __float_as_uint(fmaf(__uint_as_float(y[e]), old, __uint_as_float(v[e]) * tile));
        }
      }
#pragma unroll
      for (int e = 0; e < 16; e++) v[e] = nt > 0 && sees ? __float_as_uint(__uint_as_float(v[e]) * inv * up * part2) : 0u;
#pragma unroll
      for (int e = 0; e < 16; e += 4) *(uint4 *)(so + local * PITCH + c + e) = make_uint4(v[e], v[e + 1], v[e + 2], v[e + 3]);
    }
    tc::tc_fence_before();
  }
  __syncthreads();
  if (warp < 8 && d0 < HDP) {
    const int C = p.H * p.G * p.HD;
#pragma unroll 4
    for (int k = 0; k < PER; k++) {
      const int r = line + k * (256 / LPR);
      if (row_a + r >= nrows) break;
      const float4 v = *(const float4 *)(so + r * PITCH + d0);
      if (pp.splits > 1) {
        *(float4 *)(p.pacc + (((size_t)unit * pp.splits + split) * nrows + row_a + r) * HDP + d0) = v;
        continue;
      }
      if (d0 >= p.HD) break;
      int i, head;
      of_row(r, i, head);
      const long long orow = (long long)s * p.T + i;
      const int col = head * p.HD + d0;
      float *dst = p.out + orow * C + col;
      if (p.HD % 4 == 0) {
        *(float4 *)dst = v;
        if (p.y16) {  // (four columns lie in one group of 64)
          __half *d16 = p.y16 + ((long long)(col >> 6) * p.R + orow) * 64 + (col & 63);
          uint2 hi, lo;
          split2(v.x, v.y, hi.x, lo.x);
          split2(v.z, v.w, hi.y, lo.y);
          *(uint2 *)d16 = hi;
          if (p.lo_off) *(uint2 *)(d16 + p.lo_off) = lo;
        }
      } else {
        const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int n = 0; n < 4; n++)
          if (d0 + n < p.HD) {
            dst[n] = e[n];
            if (p.y16) {
              __half *d16 = p.y16 + ((long long)((col + n) >> 6) * p.R + orow) * 64 + ((col + n) & 63);
              const __half hi = __float2half_rn(e[n]);
              *d16 = hi;
              if (p.lo_off) d16[p.lo_off] = __float2half_rn(e[n] - __half2float(hi));
            }
          }
      }
    }
  }
  __syncthreads();
  if (gave_up && tid == 0) {
    atomicExch(p.status, kWaits + 1);
    p.status[1] = blockIdx.x, p.status[2] = 0;
  }
  if (warp == 8) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, kColumns);
  }
}

// Rows of several splits: one warp a row.
template <int HDP>
__global__ void __launch_bounds__(kThreads) k_join_kv8(const AttnParams p, int splits, int nrows, long long total) {
  fa_grid_dep_sync();
  const int lane = threadIdx.x & 31;
  const long long id = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (id >= total) return;
  const int unit = (int)(id / nrows), row = (int)(id - (long long)unit * nrows), s = unit / p.H, h = unit - s * p.H;
  Sight sight;
  bool bad;
  sight.of(p, s, bad);
  Joined<HDP> j;
  for (int k = 0; k < splits; k++) {
    const size_t part = ((size_t)unit * splits + k) * nrows + row;
    const float2 ml = *(const float2 *)(p.pml + part * 2);
    float v[HDP / 32];
#pragma unroll
    for (int i = 0; i < HDP / 32; i++) v[i] = p.pacc[part * HDP + lane + 32 * i];
    j.add(ml.x, ml.y, v);
  }
  j.finish(p, s, h, row, sight.limit(row / p.G) > 0, lane);
}

template <int HDP>
int run_prompt(fa_ctx *ctx, const fa_kv8 *c, const AttnParams &a, int most, const char *label) {
  static SmemLimit limit;
  constexpr int smem = PromptSmem<HDP>::BYTES;
  FA_CHECK_CUDA(ctx, limit.raise(ctx, k_prompt_kv8<HDP>, smem));
  PromptParams pp{};
  pp.a = a;
  const int nrows = a.G * a.T, tiles = ceil_div(most < 1 ? 1 : most, kTile);
  pp.rowtiles = ceil_div(nrows, kTile);
  const long long blocks = (long long)c->S * c->H * pp.rowtiles, slots = (long long)ctx->sm_count * (HDP <= 64 ? 2 : 1);
  // The positions are split, four tiles a split at least, while the thread blocks do not fill the GPU.  (Shorter runs of longer
  // lists even out streams of different lengths, but cost more in queries, results and joining than that gives.)
  long long splits = blocks >= slots ? 1 : slots / blocks;
  if (splits > tiles / 4) splits = tiles / 4;
  if (splits < 1) splits = 1;
  pp.per = ceil_div(tiles, (int)splits);
  pp.splits = ceil_div(tiles, pp.per);
  FA_REQUIRE(ctx, blocks * pp.splits <= 0x7fffffffLL, "%s: too many rows in one call", label);
  void *scratch = nullptr;
  size_t bytes = 0;
  const long long total = (long long)c->S * c->H * nrows;
  if (pp.splits > 1) {
    const size_t n = (size_t)total * pp.splits;
    FA_TRY(fa_block_acquire(ctx, n * (HDP + 2) * 4, &scratch, &bytes));
    pp.a.pacc = (float *)scratch, pp.a.pml = (float *)scratch + n * HDP;
  }
  int rc = FA_OK;
  cudaError_t e;
  {
    LaunchScope ls(ctx, label);
    e = fa_launch_dep(ctx, k_prompt_kv8<HDP>, dim3((unsigned)(blocks * pp.splits)), dim3(kPromptThreads), (size_t)smem, pp);
  }
  if (e == cudaSuccess && pp.splits > 1) {
    LaunchScope ls(ctx, "attn_kv8_join");
    e = fa_launch_dep(ctx, k_join_kv8<HDP>, dim3((unsigned)((total + kWarps - 1) / kWarps)), dim3(kThreads), 0, pp.a, pp.splits, nrows, total);
  }
  if (e != cudaSuccess) rc = fa_fail(ctx, FA_ERR_CUDA, "launch %s: %s", label, cudaGetErrorString(e));
  if (scratch) fa_block_release(ctx, scratch);
  return rc;
}

template <int HDP>
int run(fa_ctx *ctx, const fa_kv8 *c, AttnParams &p, int most, const char *label) {
  const int rows = p.G * p.T;
  if constexpr (HDP <= 128) {
    if (rows >= kPromptRows) return run_prompt<HDP>(ctx, c, p, most, label);
  }
  if (rows <= 4) return run<HDP, FewRows<HDP>>(ctx, c, p, most, label);
  if constexpr (HDP <= 128) {  // (16 rows of 256 do not fit the registers)
    if (rows > 8) return run<HDP, ManyRows<HDP, 2>>(ctx, c, p, most, label);
  }
  return run<HDP, ManyRows<HDP, 1>>(ctx, c, p, most, label);
}

// Attention of p's queries over the cache, whose positions end at `most` at the latest; the result is [S*T][H*G*HD].
int attend(fa_ctx *ctx, const fa_kv8 *c, AttnParams &p, int most, const char *label, fa_tensor **out) {
  fa_tensor *y = nullptr;
  const int C = c->H * p.G * c->HD;
  FA_TRY(fa_tensor_new(ctx, c->S * p.T, C, FA_F32, true, &y));
  if (y->rows == 0) {
    *out = y;
    return FA_OK;
  }
  p.out = (float *)y->dptr, p.R = y->rows;
  p.codes = c->codes, p.S = c->S, p.H = c->H, p.HD = c->HD, p.nblk = c->nblk;
  p.vec = c->HD % 4 == 0 && p.ldq % 4 == 0 && ((uintptr_t)p.q & 15) == 0;
  p.status = ctx->dev_status, p.wait_limit = ctx->wait_limit;
  if ((C & 63) == 0 && fa_tc_available(ctx)) {  // the product that follows reads the packed operand
    if (p.R <= ctx->f16_hilo_rows) {
      if ((p.y16 = fa_shadow_hilo_block(ctx, y)) != nullptr) p.lo_off = (long long)(C >> 6) * p.R * 64;
    } else {
      p.y16 = fa_shadow_block(ctx, y);
    }
    if (p.y16) y->a16_valid = true;
  }
  const int rc = c->HDP == 32 ? run<32>(ctx, c, p, most, label) : c->HDP == 64 ? run<64>(ctx, c, p, most, label)
               : c->HDP == 96 ? run<96>(ctx, c, p, most, label) : c->HDP == 128 ? run<128>(ctx, c, p, most, label)
                              : run<256>(ctx, c, p, most, label);
  if (rc != FA_OK) {
    fa_free_tensor(ctx, y);
    return rc;
  }
  *out = y;
  return FA_OK;
}

int queries(fa_ctx *ctx, const fa_kv8 *c, const fa_tensor *q, int HQ, int cols, const char *op, int *T) {
  FA_REQUIRE(ctx, fa_valid_kv8(ctx, c), "%s: unknown cache handle", op);
  FA_REQUIRE(ctx, fa_valid(ctx, q), "%s: unknown tensor handle", op);
  FA_REQUIRE(ctx, q->storage == FA_F32, "%s: operand must be f32 storage", op);
  FA_REQUIRE(ctx, HQ >= c->H && HQ % c->H == 0, "%s: %d query heads for %d key heads", op, HQ, c->H);
  FA_REQUIRE(ctx, ((long long)HQ + cols * (long long)c->H) * c->HD == q->cols, "%s: %d columns, expected %lld", op, q->cols,
             ((long long)HQ + cols * (long long)c->H) * c->HD);
  FA_REQUIRE(ctx, q->rows % c->S == 0, "%s: %d rows for %d streams", op, q->rows, c->S);
  *T = q->rows / c->S;
  FA_REQUIRE(ctx, (long long)*T * (HQ / c->H) <= 0x3fffffffLL, "%s: too many rows in one call", op);
  return fa_touch_f32(ctx, q);
}

}  // namespace

extern "C" int fa_attn_kv8(fa_ctx *ctx, const fa_tensor *q, fa_kv8 *c, int HQ, int n, const fa_tensor *lens, fa_tensor **out) {
  if (!ctx || !out) return fa_fail(ctx, FA_ERR_INVALID, "attnKv8: NULL argument");
  *out = nullptr;
  FA_CHECK_CUDA(ctx, cudaSetDevice(ctx->device));
  AttnParams p{};
  FA_TRY(queries(ctx, c, q, HQ, 0, "attnKv8", &p.T));
  FA_REQUIRE(ctx, n >= 0 && n <= c->P, "attnKv8: %d of %d positions", n, c->P);
  FA_TRY(fa_kv8_per_stream(ctx, lens, c->S, "attnKv8", "lens", &p.lens));
  p.q = (const float *)q->dptr, p.ldq = q->cols, p.G = HQ / c->H, p.n = n;
  return attend(ctx, c, p, n, "attn_kv8", out);
}

extern "C" int fa_attn_append_kv8(fa_ctx *ctx, const fa_tensor *qkv, fa_kv8 *c, int HQ, int n, const fa_tensor *pos, const fa_tensor *counts,
                                  fa_tensor **out) {
  if (!ctx || !out) return fa_fail(ctx, FA_ERR_INVALID, "attnAppendKv8: NULL argument");
  *out = nullptr;
  FA_CHECK_CUDA(ctx, cudaSetDevice(ctx->device));
  AttnParams p{};
  FA_TRY(queries(ctx, c, qkv, HQ, 2, "attnAppendKv8", &p.T));
  FA_REQUIRE(ctx, pos ? p.T <= c->P : n >= 0 && p.T <= c->P - n, "attnAppendKv8: rows %d..%lld of a cache of %d positions", n, (long long)n + p.T, c->P);
  FA_TRY(fa_kv8_per_stream(ctx, pos, c->S, "attnAppendKv8", "pos", &p.rows.pos));
  FA_TRY(fa_kv8_per_stream(ctx, counts, c->S, "attnAppendKv8", "counts", &p.rows.counts));
  p.rows.n = n, p.rows.T = p.T, p.rows.P = c->P;
  p.q = (const float *)qkv->dptr, p.ldq = qkv->cols, p.G = HQ / c->H, p.causal = 1;
  const float *k = p.q + (size_t)HQ * c->HD;
  FA_TRY(fa_kv8_write_rows(ctx, c, k, k + (size_t)c->H * c->HD, false, p.ldq, p.T, n, p.rows.pos, p.rows.counts));
  return attend(ctx, c, p, pos ? c->P : n + p.T, "attn_append_kv8", out);
}
