// Rules on logits before a token is picked: penalties for tokens of the history, a bias per token, a mask of allowed tokens.
//
//   c = how often the token occurs in the history
//   x = c > 0 ? (x > 0 ? x / repetition : x * repetition) : x
//   x = x - frequency * c - (c > 0 ? presence : 0)
//   x = x + bias
//   x = allowed ? x : -inf
// and, for a pick, the first token of the largest value among the allowed ones ({-1, -inf} where none is allowed or all are NaN).
// The reference scans a downloaded row on the host (src/engines/asr-whisper/index.ts:80-97).
//
// One pass: a cluster of thread blocks shares a row.  Each reads its part of the history once and adds to the counters of the
// block whose slice of the vocabulary a token falls into, in that block's shared memory (whole numbers: the order of the
// additions does not show), then takes its slice of the logits, whose first loads are under way meanwhile.  Every operation
// is rounded by itself, so the values are those of the formulas in f32 whatever the split.
// Bound by HBM where rows are many (4 bytes in, 4 out; the counters stay on the chip), by the latency of two cluster barriers
// and one round of loads where they are few.
#include <algorithm>
#include <type_traits>

#include "fa_internal.cuh"

namespace {

constexpr int kMaxCluster = 8;
constexpr int kBatch = 4;            // tokens of a thread at a time, and as many on their way
constexpr int kCountBytes = 196608;  // of a thread block's counts at a time
constexpr int kFew = 512, kMany = 256;  // threads of a block, see `rules`

struct LogitParams {
  const float *x;
  long long ld;
  const float *history;  // [n][S] token ids; ids outside [0, V) are no token
  int n, S, V;
  float repetition, presence, frequency;
  const float *bias;  // [1 or S] rows of bias_ld, or NULL
  long long bias_ld;
  int bias_rows;
  const uint32_t *mask;  // rows of mask_words, or NULL
  int mask_words, mask_rows;
  const float *mask_row;  // [S] or NULL
  float *out;             // [S][V] (adjust) or [S][2] (pick)
  int *status;
};

__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}

__device__ __forceinline__ uint32_t in_block(const void *p, uint32_t rank) {  // the same shared variable in block `rank` of the cluster
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  return a;
}

// n floats from p on into L2, but for what lies outside whole 16-byte groups.
__device__ __forceinline__ void to_l2(const float *p, int n) {
  const uintptr_t from = ((uintptr_t)p + 15) & ~(uintptr_t)15, to = (uintptr_t)(p + n) & ~(uintptr_t)15;
  if (n > 0 && to > from) asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(from), "r"((uint32_t)(to - from)) : "memory");
}

// PICK: the best token instead of the logits; HISTORY, BIAS, MASK: which rules there are.  HISTORY 1 counts in 16 bits (fewer
// than 65536 tokens), 2 in 32.
template <int kThreads, bool PICK, int HISTORY, bool BIAS, bool MASK>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) k_adjust(const LogitParams p) {
  using Count = std::conditional_t<HISTORY == 1, uint16_t, uint32_t>;
  constexpr int kSlice = kCountBytes / (int)sizeof(Count);
  extern __shared__ uint32_t words[];
  const Count *cnt = (const Count *)words;  // one slice's counts
  __shared__ float bv[kThreads / 32];
  __shared__ int bi[kThreads / 32];
  __shared__ float cv;  // this block's best, read by rank 0
  __shared__ int ci;
  fa_grid_dep_sync();
  const int nc = (int)cluster_size(), rank = (int)cluster_rank(), s = blockIdx.x / nc;
  const float *row = p.x + (long long)s * p.ld;
  const float *bias = BIAS ? p.bias + (p.bias_rows > 1 ? (long long)s * p.bias_ld : 0) : nullptr;
  const uint32_t *mask = nullptr;
  if (MASK) {
    int r = p.mask_rows > 1 ? s : 0;
    if (p.mask_row) {
      const float f = p.mask_row[s];
      const bool fits = f >= 0.0f && f < (float)p.mask_rows;
      if (!fits && rank == 0 && threadIdx.x == 0) atomicOr(p.status + 3, kStatusMaskRow);
      r = fits ? (int)f : 0;
    }
    mask = p.mask + (long long)r * p.mask_words;
  }
  float best = -INFINITY;
  int at = 0x7fffffff;
  const int width = ((p.V + nc - 1) / nc + 31) / 32 * 32, v1 = min(p.V, (rank + 1) * width);
  for (int off = 0; off < width; off += kSlice) {  // (every block of the cluster: they count for one another)
    const int a = min(p.V, rank * width + off), b = min(v1, a + kSlice);
    // a thread takes j0, j0 + kThreads, ...: a warp's 32 neighbours share a word of the mask, each its lane's bit
    const float *px = row + a + threadIdx.x, *pb = BIAS ? bias + a + threadIdx.x : nullptr;
    const uint32_t *pm = MASK ? mask + ((a + (int)threadIdx.x) >> 5) : nullptr;
    float *po = PICK ? nullptr : p.out + (long long)s * p.V + a + threadIdx.x;
    float x[kBatch], bb[BIAS ? kBatch : 1];
    uint32_t w[MASK ? kBatch : 1];
    if (threadIdx.x == 0) {  // the slice on its way to L2 while the history is counted
      to_l2(row + a, b - a);
      if (BIAS) to_l2(bias + a, b - a);
    }
    int left = b - a - (int)threadIdx.x, k = threadIdx.x;  // tokens from this thread's on, place in the slice
    auto load = [&]() {
      if (left > (kBatch - 1) * kThreads) {
#pragma unroll
        for (int u = 0; u < kBatch; u++) {
          x[u] = __ldcs(px + u * kThreads);
          if (BIAS) bb[u] = __ldcs(pb + u * kThreads);
          if (MASK) w[u] = pm[u * (kThreads / 32)];
        }
      } else {
#pragma unroll
        for (int u = 0; u < kBatch; u++) {
          const bool in = u * kThreads < left;
          x[u] = in ? __ldcs(px + u * kThreads) : 0.0f;
          if (BIAS) bb[u] = in ? pb[u * kThreads] : 0.0f;
          if (MASK) w[u] = in ? pm[u * (kThreads / 32)] : 0u;
        }
      }
      px += kBatch * kThreads;
      if (BIAS) pb += kBatch * kThreads;
      if (MASK) pm += kBatch * (kThreads / 32);
    };
    load();
    if (HISTORY) {
      for (int i = threadIdx.x; i < min(width, kSlice) / (4 / (int)sizeof(Count)); i += kThreads) words[i] = 0;
      cluster_sync();
      const int i0 = (int)((long long)p.n * rank / nc), i1 = (int)((long long)p.n * (rank + 1) / nc);
      for (int i = i0 + threadIdx.x; i < i1; i += kThreads) {
        const float f = p.history[(long long)i * p.S + s];
        if (!(f >= 0.0f && f < (float)p.V)) continue;
        const int token = (int)f, owner = token / width, c = token - owner * width - off;
        if (c >= 0 && c < kSlice)
          asm volatile("red.relaxed.cluster.shared::cluster.add.u32 [%0], %1;" ::"r"(in_block(words + (HISTORY == 1 ? c >> 1 : c), owner)),
                       "r"(HISTORY == 1 && (c & 1) ? 65536u : 1u)
                       : "memory");
      }
      cluster_sync();
    }
    auto step = [&](int u, float y, float add, uint32_t word) {
      if (HISTORY) {
        const uint32_t c = cnt[k + u * kThreads];
        if (c) {
          y = y > 0.0f ? __fdiv_rn(y, p.repetition) : __fmul_rn(y, p.repetition);
          y = __fsub_rn(__fsub_rn(y, __fmul_rn((float)c, p.frequency)), p.presence);
        }
      }
      if (BIAS) y = __fadd_rn(y, add);
      const bool allowed = !MASK || (word >> (threadIdx.x & 31) & 1u);
      if (PICK) {
        if (allowed && (y > best || (y == best && a + k + u * kThreads < at))) best = y, at = a + k + u * kThreads;  // (a NaN never wins)
      } else {
        __stcs(po + u * kThreads, allowed ? y : -INFINITY);
      }
    };
    while (left > 0) {
      float y[kBatch], add[BIAS ? kBatch : 1];
      uint32_t word[MASK ? kBatch : 1];
#pragma unroll
      for (int u = 0; u < kBatch; u++) {
        y[u] = x[u];
        if (BIAS) add[u] = bb[u];
        if (MASK) word[u] = w[u];
      }
      const int now = left;
      left -= kBatch * kThreads;
      if (left > 0) load();
#pragma unroll
      for (int u = 0; u < kBatch; u++)
        if (u * kThreads < now) step(u, y[u], BIAS ? add[BIAS ? u : 0] : 0.0f, MASK ? word[MASK ? u : 0] : 0u);
      k += kBatch * kThreads;
      if (!PICK) po += kBatch * kThreads;
    }
    if (HISTORY && off + kSlice < width) cluster_sync();  // (the counts are read)
  }
  if (!PICK) return;
  auto take = [&](float v, int j) {
    if (v > best || (v == best && j < at)) best = v, at = j;
  };
  auto warp_best = [&]() {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float v = __shfl_xor_sync(0xffffffffu, best, o);
      take(v, __shfl_xor_sync(0xffffffffu, at, o));
    }
  };
  warp_best();
  if ((threadIdx.x & 31) == 0) bv[threadIdx.x >> 5] = best, bi[threadIdx.x >> 5] = at;
  __syncthreads();
  if (threadIdx.x < 32) {
    best = bv[threadIdx.x & (kThreads / 32 - 1)], at = bi[threadIdx.x & (kThreads / 32 - 1)];
    warp_best();
    if (threadIdx.x == 0) cv = best, ci = at;
  }
  if (nc > 1) {
    cluster_sync();
    if (rank == 0 && threadIdx.x < 32) {
      const uint32_t r = threadIdx.x & (nc - 1);
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(best) : "r"(in_block(&cv, r)) : "memory");
      asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(at) : "r"(in_block(&ci, r)) : "memory");
      warp_best();
    }
  }
  if (rank == 0 && threadIdx.x == 0) {
    p.out[2 * (long long)s] = at == 0x7fffffff ? -1.0f : (float)at;
    p.out[2 * (long long)s + 1] = best;
  }
  if (nc > 1) cluster_sync();  // no block leaves while its result is read
}

int rules(fa_ctx *ctx, const fa_tensor *x, int ncols, const fa_logit_rules *r, bool pick, fa_tensor **out) {
  const char *op = pick ? "pickAdjusted" : "adjustLogits";
  if (!ctx || !out || !r) return fa_fail(ctx, FA_ERR_INVALID, "%s: NULL argument", op);
  *out = nullptr;
  FA_CHECK_CUDA(ctx, cudaSetDevice(ctx->device));
  auto f32 = [&](const fa_tensor *t) {
    FA_REQUIRE(ctx, fa_valid(ctx, t), "%s: unknown tensor handle", op);
    FA_REQUIRE(ctx, t->storage == FA_F32, "%s: operand must be f32 storage", op);
    return fa_touch_f32(ctx, t);
  };
  FA_TRY(f32(x));
  FA_REQUIRE(ctx, x->cols > 0 && ncols <= x->cols, "%s: %d of %d columns", op, ncols, x->cols);
  LogitParams p{};
  p.S = x->rows, p.V = ncols > 0 ? ncols : x->cols, p.ld = x->cols, p.x = (const float *)x->dptr;
  FA_REQUIRE(ctx, p.V <= (1 << 24), "%s: %d columns: token ids are f32 values, 2^24 at most", op, p.V);
  if (r->history) {
    FA_TRY(f32(r->history));
    FA_REQUIRE(ctx, r->history->cols == p.S, "%s: the history has %d columns for %d rows of logits", op, r->history->cols, p.S);
    FA_REQUIRE(ctx, r->n >= 0 && r->n <= r->history->rows, "%s: %d of %d history rows", op, r->n, r->history->rows);
    FA_REQUIRE(ctx, r->repetition > 0.0f && r->repetition < INFINITY, "%s: repetition penalty %g", op, (double)r->repetition);
    if (r->n && (r->repetition != 1.0f || r->presence != 0.0f || r->frequency != 0.0f)) p.history = (const float *)r->history->dptr, p.n = r->n;
  }
  p.repetition = r->repetition, p.presence = r->presence, p.frequency = r->frequency;
  if (r->bias) {
    FA_TRY(f32(r->bias));
    FA_REQUIRE(ctx, r->bias->cols >= p.V && (r->bias->rows == 1 || r->bias->rows == p.S), "%s: bias is %dx%d, expected 1 or %d rows of %d", op,
               r->bias->rows, r->bias->cols, p.S, p.V);
    p.bias = (const float *)r->bias->dptr, p.bias_ld = r->bias->cols, p.bias_rows = r->bias->rows;
  }
  if (r->mask) {
    FA_REQUIRE(ctx, fa_valid_bytes(ctx, r->mask), "%s: unknown mask handle", op);
    p.mask_words = ceil_div(p.V, 32);
    const size_t rows = r->mask->nbytes / ((size_t)p.mask_words * 4);
    FA_REQUIRE(ctx, rows >= 1 && rows <= (1 << 24) && r->mask->nbytes == rows * p.mask_words * 4, "%s: mask of %zu bytes is no whole number of rows of %d", op,
               r->mask->nbytes, p.mask_words * 4);
    p.mask_rows = (int)rows, p.mask = (const uint32_t *)r->mask->dptr;
    if (r->mask_rows) {
      FA_TRY(f32(r->mask_rows));
      FA_REQUIRE(ctx, (long long)r->mask_rows->rows * r->mask_rows->cols == p.S, "%s: maskRows needs %d values", op, p.S);
      p.mask_row = (const float *)r->mask_rows->dptr;
    } else {
      FA_REQUIRE(ctx, p.mask_rows == 1 || p.mask_rows == p.S, "%s: %d mask rows for %d rows of logits: say which with maskRows", op, p.mask_rows, p.S);
    }
  } else {
    FA_REQUIRE(ctx, !r->mask_rows, "%s: maskRows without a mask", op);
  }
  fa_tensor *y = nullptr;
  FA_TRY(fa_tensor_new(ctx, p.S, pick ? 2 : p.V, FA_F32, true, &y));
  if (p.S) {
    p.out = (float *)y->dptr, p.status = ctx->dev_status;
    // Blocks of a row: as many as one wave of two blocks an SM takes, and so many that a block's tokens are at most 16640.  The
    // two shapes of a block, us, 512 threads (two an SM) / 256 (four): one row of 51866 tokens, pick 6.4 / 7.4; 64 rows 10.3 /
    // 14.7; 256 rows of 131075, values 127 / 114, pick 148 / 121.  More threads an SM of either shape are slower for many rows
    // (256 x 6: 145): the loads of one batch wait behind the others'.
    int nc = 1;
    while (nc < kMaxCluster && p.V > nc * 2048 && (p.S * nc <= ctx->sm_count || p.V > nc * 16640)) nc *= 2;
    const int width = (int)round_up(ceil_div(p.V, nc), 32);
    const int counts = !p.history ? 0 : p.n < 65536 ? 1 : 2;
    const bool few = (long long)p.S * nc <= 2 * ctx->sm_count || counts == 2;
    const size_t smem = counts ? std::min<size_t>((size_t)width * (counts == 1 ? 2 : 4), kCountBytes) : 0;
    using Kernel = void (*)(LogitParams);
#define FORMS(THREADS, PICK, HISTORY)                                                                        \
  {k_adjust<THREADS, PICK, HISTORY, false, false>, k_adjust<THREADS, PICK, HISTORY, false, true>,            \
   k_adjust<THREADS, PICK, HISTORY, true, false>, k_adjust<THREADS, PICK, HISTORY, true, true>}
#define ROWS(PICK) {FORMS(kMany, PICK, 0), FORMS(kMany, PICK, 1), FORMS(kFew, PICK, 0), FORMS(kFew, PICK, 1), FORMS(kFew, PICK, 2)}
    static const Kernel kernels[2][5][4] = {ROWS(false), ROWS(true)};
#undef ROWS
#undef FORMS
    static SmemLimit limit[2][5][4];
    const int form = few ? 2 + counts : counts;
    const int which = (p.bias ? 2 : 0) + (p.mask ? 1 : 0);
    const Kernel kernel = kernels[pick][form][which];
    cudaError_t e = p.history ? limit[pick][form][which].raise(ctx, kernel, kCountBytes) : cudaSuccess;
    if (e == cudaSuccess) {
      LaunchScope ls(ctx, pick ? "pick_adjusted" : "adjust_logits");
      cudaLaunchConfig_t cfg{};
      cfg.gridDim = dim3((unsigned)(p.S * nc)), cfg.blockDim = dim3(few ? kFew : kMany), cfg.dynamicSmemBytes = smem, cfg.stream = ctx->stream;
      cudaLaunchAttribute attr[2];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = nc, attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
      attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
      attr[1].val.programmaticStreamSerializationAllowed = ctx->pdl ? 1 : 0;
      cfg.attrs = attr, cfg.numAttrs = 2;
      e = cudaLaunchKernelEx(&cfg, kernel, p);
    }
    if (e != cudaSuccess) {
      fa_free_tensor(ctx, y);
      return fa_fail(ctx, FA_ERR_CUDA, "launch %s: %s", op, cudaGetErrorString(e));
    }
  }
  *out = y;
  return FA_OK;
}

}  // namespace

extern "C" int fa_adjust_logits(fa_ctx *ctx, const fa_tensor *x, int ncols, const fa_logit_rules *r, fa_tensor **out) {
  return rules(ctx, x, ncols, r, false, out);
}
extern "C" int fa_pick_adjusted(fa_ctx *ctx, const fa_tensor *x, int ncols, const fa_logit_rules *r, fa_tensor **out) {
  return rules(ctx, x, ncols, r, true, out);
}
