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
// One pass: a cluster of thread blocks shares a row, each block counts the history's tokens that fall into its slice of the
// vocabulary in shared memory (whole numbers: the order of the atomics does not show) and then reads its slice of the logits
// once.  Every operation is rounded by itself, so the values are those of the formulas in f32 whatever the split.
#include "fa_internal.cuh"

namespace {

constexpr int kThreads = 512, kMaxCluster = 8, kSlice = 16384;  // tokens that a thread block counts at a time (32 KB)

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

template <bool PICK>
__global__ void __launch_bounds__(kThreads) k_adjust(const LogitParams p) {
  extern __shared__ uint32_t cnt[];  // one slice's counts
  __shared__ float bv[kThreads / 32];
  __shared__ int bi[kThreads / 32];
  __shared__ float cv;  // this block's best, read by rank 0
  __shared__ int ci;
  fa_grid_dep_sync();
  const int nc = (int)cluster_size(), rank = (int)cluster_rank(), s = blockIdx.x / nc;
  const float *row = p.x + (long long)s * p.ld;
  const float *bias = p.bias ? p.bias + (p.bias_rows > 1 ? (long long)s * p.bias_ld : 0) : nullptr;
  const uint32_t *mask = nullptr;
  if (p.mask) {
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
  const int width = ((p.V + nc - 1) / nc + 31) / 32 * 32, v0 = min(p.V, rank * width), v1 = min(p.V, v0 + width);
  for (int a = v0; a < v1; a += kSlice) {
    const int b = min(v1, a + kSlice);
    if (p.history) {
      for (int i = threadIdx.x; i < b - a; i += kThreads) cnt[i] = 0;
      __syncthreads();
      for (int i = threadIdx.x; i < p.n; i += kThreads) {
        const float f = p.history[(long long)i * p.S + s];
        if (f >= (float)a && f < (float)b) atomicAdd(&cnt[(int)f - a], 1u);
      }
      __syncthreads();
    }
    for (int j = a + threadIdx.x; j < b; j += kThreads) {
      float x = row[j];
      if (p.history) {
        const uint32_t c = cnt[j - a];
        if (c) {
          x = x > 0.0f ? __fdiv_rn(x, p.repetition) : __fmul_rn(x, p.repetition);
          x = __fsub_rn(__fsub_rn(x, __fmul_rn((float)c, p.frequency)), p.presence);
        }
      }
      if (bias) x = __fadd_rn(x, bias[j]);
      const bool allowed = !mask || (mask[j >> 5] >> (j & 31) & 1u);
      if (PICK) {
        if (allowed && (x > best || (x == best && j < at))) best = x, at = j;  // (a NaN never wins)
      } else {
        p.out[(long long)s * p.V + j] = allowed ? x : -INFINITY;
      }
    }
    __syncthreads();
  }
  if (!PICK) return;
  auto take = [&](float v, int j) {
    if (v > best || (v == best && j < at)) best = v, at = j;
  };
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float v = __shfl_xor_sync(0xffffffffu, best, o);
    take(v, __shfl_xor_sync(0xffffffffu, at, o));
  }
  if ((threadIdx.x & 31) == 0) bv[threadIdx.x >> 5] = best, bi[threadIdx.x >> 5] = at;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kThreads / 32; w++) take(bv[w], bi[w]);
    cv = best, ci = at;
  }
  cluster_sync();
  if (rank == 0 && threadIdx.x == 0) {
    for (int r = 1; r < nc; r++) {
      float v;
      int j;
      uint32_t addr_v, addr_j;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr_v) : "r"((uint32_t)__cvta_generic_to_shared(&cv)), "r"(r));
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr_j) : "r"((uint32_t)__cvta_generic_to_shared(&ci)), "r"(r));
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr_v) : "memory");
      asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(j) : "r"(addr_j) : "memory");
      take(v, j);
    }
    p.out[2 * s] = at == 0x7fffffff ? -1.0f : (float)at;
    p.out[2 * s + 1] = best;
  }
  cluster_sync();  // no block leaves while its result is read
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
    int nc = 1;
    while (nc < kMaxCluster && (long long)p.S * nc < 2 * ctx->sm_count && p.V > nc * 2048) nc *= 2;
    const int width = (int)round_up(ceil_div(p.V, nc), 32);
    const size_t smem = p.history ? (size_t)4 * (width < kSlice ? width : kSlice) : 0;
    static SmemLimit limit[2];
    auto kernel = pick ? k_adjust<true> : k_adjust<false>;
    cudaError_t e = limit[pick].raise(ctx, kernel, kSlice * 4);
    if (e == cudaSuccess) {
      LaunchScope ls(ctx, pick ? "pick_adjusted" : "adjust_logits");
      cudaLaunchConfig_t cfg{};
      cfg.gridDim = dim3((unsigned)(p.S * nc)), cfg.blockDim = dim3(kThreads), cfg.dynamicSmemBytes = smem, cfg.stream = ctx->stream;
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
