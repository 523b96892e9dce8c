// Attention over the 8-bit key and value cache (fa_kv8.cuh): out = sum_j p_j v_j / sum_j p_j, p_j = exp(q.k_j - max).
//
// Rows: the G = HQ / H query heads that share a key head times the T queries of a stream, row r = query r / G, head r % G.
//
// Arithmetic.  Codes are whole numbers of 8 bits, so they are exact in f16; the other side of each product is split into an
// f16 value and its f16 residue (22 bits and more), the two sitting in the upper and lower 8 rows of ONE m16n8k16 product, so
// that a warp's product serves 8 rows with f32-grade operands and f32 sums.  A query row is scaled by a power of two to
// [1, 2) before the split and the block's scale multiplies the sums afterwards.  Weights are exp(s - the block's own row
// maximum), so that the largest is 1 whatever the other blocks hold; what the block then adds to the running result is scaled
// by exp(block maximum - running maximum) times the values' scale, in f32.
#include "fa_kv8.cuh"
#include "fa_tc_common.cuh"

namespace {

using kv8::kBlock;
using tc::smem_u32;

constexpr int kWarps = 4, kThreads = kWarps * 32;

struct AttnParams {
  const float *q;  // query row i of stream s, head h: q + (s*T + i)*ldq + h*HD
  long long ldq;
  const uint8_t *codes;
  const float *lens;  // [S] on the device, or NULL: n for all (complete caches)
  kv8::Rows rows;     // causal: where the queries stand
  int causal, n;
  int H, G, T, HD, nblk, vec;
  int rowgroups, splits, kper;  // row groups of a unit, its splits and their blocks
  float *out;                   // [S*T][H*G*HD]
  __half *y16;                  // packed f16 row operand of out (value plane, then residue plane), or NULL
  long long lo_off;
  int R;                        // rows of out
  float *pacc, *pml;            // splits > 1: [unit][rowgroup][split][8*RG][HDP] and [..][8*RG][2]
  int *tickets;
  int *status;
  unsigned wait_limit;
};

__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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
// Four codes u to two pairs of f16 u - 128: 0x6400 | u is 1024 + u.
__device__ __forceinline__ void widen(uint32_t w, uint32_t &b0, uint32_t &b1) {
  const __half2 bias = __half2half2(__ushort_as_half(0x6480));  // 1152
  const uint32_t x = __byte_perm(w, 0x64646464u, 0x4140), y = __byte_perm(w, 0x64646464u, 0x4342);
  const __half2 p = __hsub2(*(const __half2 *)&x, bias), q = __hsub2(*(const __half2 *)&y, bias);
  b0 = *(const uint32_t *)&p, b1 = *(const uint32_t *)&q;
}
// exp(m - M) for M >= m, 1 where the two are the same infinity
__device__ __forceinline__ float rescale(float m, float M) { return m == M ? 1.0f : __expf(m - M); }

template <int HDP>
__host__ __device__ constexpr int stages() { return HDP <= 32 ? 6 : HDP <= 64 ? 4 : HDP <= 128 ? 3 : 2; }

// One warp per block of 32 positions; a thread block = one (stream, head), one group of 8*RG rows, one split of the blocks,
// which its four warps take in turn, each through a ring of its own that the copy engine fills.
template <int HDP, int RG>
__global__ void __launch_bounds__(kThreads) k_attn_kv8(const AttnParams p) {
  constexpr int KS = HDP / 16, NT = HDP / 8, BB = (int)kv8::block_bytes(HDP), NST = stages<HDP>(), ROWS = 8 * RG;
  extern __shared__ __align__(128) uint8_t ring[];  // [kWarps][NST][BB]; the warps' results afterwards
  __shared__ __align__(8) uint64_t full[kWarps][NST];
  __shared__ float sml[kWarps][ROWS][2];
  __shared__ int last;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  uint32_t blk = blockIdx.x;
  const int split = blk % p.splits;
  blk /= p.splits;
  const int rg = blk % p.rowgroups, unit = blk / p.rowgroups, s = unit / p.H, h = unit - s * p.H;
  const int nrows = p.G * p.T;
  if (threadIdx.x < kWarps * NST) tc::mbar_init(smem_u32(&full[0][0] + threadIdx.x), 1);
  tc::fence_barrier_init();
  __syncthreads();
  fa_grid_dep_sync();

  // how far this group's rows see
  int start = 0, count = p.T, len = p.n;
  bool bad = false;
  if (p.causal) p.rows.of(s, start, count, bad);
  else if (p.lens) {
    const float f = p.lens[s];
    bad = !(f >= 0.0f && f <= (float)p.n);
    len = f >= 0.0f ? (int)fminf(f, (float)p.n) : 0;
  }
  if (bad && threadIdx.x == 0) atomicOr(p.status + 3, kStatusKv8Length);
  auto limit = [&](int row) {
    if (row >= nrows) return 0;
    const int i = row / p.G;
    return !p.causal ? len : i < count ? start + i + 1 : 0;
  };
  const int top_row = min(nrows, (rg + 1) * ROWS) - 1;
  const int most = p.causal ? (min(top_row / p.G, count - 1) >= rg * ROWS / p.G ? start + min(top_row / p.G, count - 1) + 1 : 0) : len;
  const int nb = (most + kBlock - 1) / kBlock, b0 = split * p.kper + warp, b1 = min(nb, (split + 1) * p.kper);

  // ring: this warp's blocks b0, b0 + 4, ...
  const uint8_t *src = p.codes + (size_t)unit * p.nblk * BB;
  const uint32_t mine = smem_u32(ring) + warp * (NST * BB), bars = smem_u32(&full[warp][0]);
  auto fetch = [&](int b, int st) {
    tc::mbar_expect_tx(bars + 8 * st, BB);
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(mine + st * BB),
                 "l"(src + (size_t)b * BB), "r"(BB), "r"(bars + 8 * st)
                 : "memory");
  };
  if (lane == 0)
    for (int k = 0; k < NST; k++)
      if (b0 + k * kWarps < b1) fetch(b0 + k * kWarps, k);

  // query rows as f16 value and residue, scaled to [1, 2)
  uint32_t qf[RG][KS][4];
  float qs[RG], m[RG], l[RG], o[RG][NT][2];
  int lim[RG];
#pragma unroll
  for (int r = 0; r < RG; r++) {
    const int row = rg * ROWS + r * 8 + g;
    lim[r] = limit(row);
    m[r] = -INFINITY, l[r] = 0.0f;
#pragma unroll
    for (int i = 0; i < NT; i++) o[r][i][0] = o[r][i][1] = 0.0f;
    const int rr = min(row, nrows - 1), i = rr / p.G;
    const float *qp = p.q + ((long long)s * p.T + i) * p.ldq + (h * p.G + rr - i * p.G) * p.HD;
    float x[KS][4], a = 0.0f;
    bool nan = false;
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
#pragma unroll
      for (int e = 0; e < 4; e++) a = fmaxf(a, fabsf(x[k][e])), nan |= x[k][e] != x[k][e];
    }
    a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 1));
    a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 2));
    const uint32_t quad = 15u << (lane & 28);
    nan = (__ballot_sync(0xffffffffu, nan) & quad) != 0;
    int ex = __float_as_int(a) >> 23;  // a >= 0
    const bool finite = ex < 255 && !nan;
    ex = min(max(ex, 1), 253);
    qs[r] = finite ? __int_as_float(ex << 23) * 1.0f : __int_as_float(0x7fc00000);  // 2^(ex - 127); NaN scores for a row that is not finite
    const float f = finite ? __int_as_float((254 - ex) << 23) : 0.0f;
#pragma unroll
    for (int k = 0; k < KS; k++) {
      if (!finite) x[k][0] = x[k][1] = x[k][2] = x[k][3] = 0.0f;
      split2(x[k][0] * f, x[k][1] * f, qf[r][k][0], qf[r][k][1]);
      split2(x[k][2] * f, x[k][3] * f, qf[r][k][2], qf[r][k][3]);
    }
  }

  bool ok = true;
  int st = 0, parity = 0;
  for (int b = b0; b < b1; b += kWarps) {
    ok = __all_sync(0xffffffffu, tc::mbar_wait(bars + 8 * st, parity, p.wait_limit)) && ok;
    const uint8_t *sb = ring + warp * (NST * BB) + st * BB;
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
#pragma unroll
        for (int r = 0; r < RG; r++) mma(sc[r][(4 * c + u) / KS], qf[r][(4 * c + u) % KS], x, y);
      }
    }
    const float2 scales = *(const float2 *)(sb + 2 * kBlock * HDP);
    uint32_t pf[RG][2][4];
    float add[RG], old[RG];
    bool sees[RG];
#pragma unroll
    for (int r = 0; r < RG; r++) {
      const int n = lim[r] - b * kBlock - 8 * t;  // this lane's positions 0..n-1 are seen
      float v[4][2], top = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; j++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          v[j][e] = (sc[r][j][e] + sc[r][j][2 + e]) * qs[r] * scales.x;
          if (2 * j + e < n) top = fmaxf(top, v[j][e]);
        }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const float ref = top == -INFINITY ? 0.0f : top;
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; j++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          v[j][e] = 2 * j + e < n ? __expf(v[j][e] - ref) : 0.0f;
          sum += v[j][e];
        }
      const float M = fmaxf(m[r], top);
      sees[r] = lim[r] > b * kBlock;
      old[r] = rescale(m[r], M);
      const float c = rescale(top, M);
      if (sees[r]) l[r] = l[r] * old[r] + sum * c;
      add[r] = c * scales.y;
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
          mma(acc, pf[r][0], x0, y0);
          mma(acc, pf[r][1], x1, y1);
          float(&d)[2] = o[r][2 * c + u];
          if (sees[r]) {
            d[0] = fmaf(d[0], old[r], (acc[0] + acc[2]) * add[r]);
            d[1] = fmaf(d[1], old[r], (acc[1] + acc[3]) * add[r]);
          }
        }
      }
    }
    __syncwarp();
    if (lane == 0 && b + NST * kWarps < b1) fetch(b + NST * kWarps, st);
    if (++st == NST) st = 0, parity ^= 1;
  }
  if (!ok && lane == 0) {
    atomicExch(p.status, 81);
    p.status[1] = blockIdx.x, p.status[2] = warp;
  }

  // the four warps' results, then the splits'
  float *mo = (float *)(ring + warp * (NST * BB));  // [ROWS][HDP]
#pragma unroll
  for (int r = 0; r < RG; r++) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    if (t == 0) sml[warp][r * 8 + g][0] = m[r], sml[warp][r * 8 + g][1] = l[r];
#pragma unroll
    for (int i = 0; i < NT; i++) *(float2 *)(mo + (r * 8 + g) * HDP + 8 * i + 2 * t) = make_float2(o[r][i][0], o[r][i][1]);
  }
  __syncthreads();
  auto finish = [&](int row, int d, float M, float L, float a) {  // one value of the result
    const int gr = rg * ROWS + row;
    if (gr >= nrows || d >= p.HD) return;
    const int i = gr / p.G, col = (h * p.G + gr - i * p.G) * p.HD + d, C = p.H * p.G * p.HD;
    const float y = limit(gr) > 0 ? a / L : 0.0f;
    const long long orow = (long long)s * p.T + i;
    p.out[orow * C + col] = y;
    if (p.y16) {
      __half *d16 = p.y16 + ((long long)(col >> 6) * p.R + orow) * 64 + (col & 63);
      const __half hi = __float2half_rn(y);
      *d16 = hi;
      if (p.lo_off) d16[p.lo_off] = __float2half_rn(y - __half2float(hi));
    }
  };
  const size_t part = ((size_t)unit * p.rowgroups + rg) * p.splits;
  for (int i = threadIdx.x; i < ROWS * HDP; i += kThreads) {
    const int row = i / HDP, d = i - row * HDP;
    float M = -INFINITY, L = 0.0f, a = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; w++) M = fmaxf(M, sml[w][row][0]);
#pragma unroll
    for (int w = 0; w < kWarps; w++) {
      const float f = rescale(sml[w][row][0], M);
      L += sml[w][row][1] * f;
      a += *((const float *)(ring + w * (NST * BB)) + i) * f;
    }
    if (p.splits == 1) {
      finish(row, d, M, L, a);
    } else {
      p.pacc[(part + split) * ROWS * HDP + i] = a;
      if (d == 0) *(float2 *)(p.pml + ((part + split) * ROWS + row) * 2) = make_float2(M, L);
    }
  }
  if (p.splits == 1) return;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    int *tk = p.tickets + (size_t)unit * p.rowgroups + rg;
    last = atomicAdd(tk, 1) == p.splits - 1;
    if (last) *tk = 0;  // ready for the next launch on this stream
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  for (int i = threadIdx.x; i < ROWS * HDP; i += kThreads) {
    const int row = i / HDP, d = i - row * HDP;
    float M = -INFINITY, L = 0.0f, a = 0.0f;
    for (int k = 0; k < p.splits; k++) M = fmaxf(M, __ldcg(p.pml + ((part + k) * ROWS + row) * 2));
    for (int k = 0; k < p.splits; k++) {
      const float2 ml = __ldcg((const float2 *)(p.pml + ((part + k) * ROWS + row) * 2));
      const float f = rescale(ml.x, M);
      L += ml.y * f;
      a += __ldcg(p.pacc + (part + k) * ROWS * HDP + i) * f;
    }
    finish(row, d, M, L, a);
  }
}

template <int HDP, int RG>
cudaError_t launch(fa_ctx *ctx, const AttnParams &p, int grid) {
  static SmemLimit limit;
  constexpr size_t smem = (size_t)kWarps * stages<HDP>() * kv8::block_bytes(HDP);
  const cudaError_t e = limit.raise(ctx, k_attn_kv8<HDP, RG>, smem);
  if (e != cudaSuccess) return e;
  return fa_launch_dep(ctx, k_attn_kv8<HDP, RG>, dim3(grid), dim3(kThreads), smem, p);
}
template <int HDP>
cudaError_t launch(fa_ctx *ctx, const AttnParams &p, int rgroups, int grid) {
  return rgroups == 1 ? launch<HDP, 1>(ctx, p, grid) : launch<HDP, 2>(ctx, p, grid);
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
  p.codes = c->codes, p.H = c->H, p.HD = c->HD, p.nblk = c->nblk;
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
  const int rgroup = p.G * p.T > 8 && c->HDP <= 128 ? 2 : 1, nb = ceil_div(most < 1 ? 1 : most, kBlock);
  p.rowgroups = ceil_div(p.G * p.T, 8 * rgroup);
  const long long units = (long long)c->S * c->H * p.rowgroups;
  long long splits = (4ll * ctx->sm_count + units - 1) / units;
  if (splits > ceil_div(nb, kWarps)) splits = ceil_div(nb, kWarps);
  if (units > ctx->gemv_ticket_count) splits = 1;
  p.kper = ceil_div(ceil_div(nb, (int)splits), kWarps) * kWarps;
  p.splits = ceil_div(nb, p.kper);
  void *scratch = nullptr;
  size_t bytes = 0;
  int rc = FA_OK;
  if (units * p.splits > 0x7fffffffLL) rc = fa_fail(ctx, FA_ERR_INVALID, "%s: too many rows in one call", label);
  if (rc == FA_OK && p.splits > 1) {
    const size_t n = (size_t)units * p.splits * 8 * rgroup;
    rc = fa_block_acquire(ctx, n * c->HDP * 4 + n * 8, &scratch, &bytes);
    p.pacc = (float *)scratch, p.pml = (float *)scratch + n * c->HDP, p.tickets = ctx->gemv_tickets;
  }
  if (rc == FA_OK) {
    LaunchScope ls(ctx, label);
    const int grid = (int)(units * p.splits);
    const cudaError_t e = c->HDP == 32 ? launch<32>(ctx, p, rgroup, grid) : c->HDP == 64 ? launch<64>(ctx, p, rgroup, grid)
                        : c->HDP == 96 ? launch<96>(ctx, p, rgroup, grid) : c->HDP == 128 ? launch<128>(ctx, p, rgroup, grid)
                                       : launch<256, 1>(ctx, p, grid);
    if (e != cudaSuccess) rc = fa_fail(ctx, FA_ERR_CUDA, "launch %s: %s", label, cudaGetErrorString(e));
  }
  if (scratch) fa_block_release(ctx, scratch);
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
