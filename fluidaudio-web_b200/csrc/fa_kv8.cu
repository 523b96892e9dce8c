// The 8-bit key and value cache: its handle, the kernel that codes rows into it and the one that reads them back.
//
// The decoder's cross-attention reads every key and value of a clip once per token: 983 MB per layer for 64 streams in f32
// (src/engines/asr-whisper/raw-whisper-decoder.js:126-131 reads the same tensors).  In 8 bits with a scale for each block of
// 32 positions and head it is 246 MB.
//
// What a cache holds depends on its rows alone, not on how they came: the block that is not full yet is coded from its f32
// rows (kept in `tail`) again whenever a row joins it, so appending one by one and writing all at once store the same codes.
// A call that goes back to an earlier block than the last one written takes that block's rows at their stored values.
#include "fa_kv8.cuh"

namespace {

using kv8::kBlock;

constexpr int kThreads = 128;

struct WriteParams {
  const void *src[2];  // keys, values: row (s, i) of head h at src + (s*T + i)*ld + h*HD
  long long ld;
  uint8_t *codes;
  float *tail;
  int *tag;
  kv8::Rows rows;
  int H, HD, HDP, nblk;
  int vec;  // rows may be read four values at a time
  int *status;
};

// rint(x / scale), the quotient exact where it matters: the product with 1 / scale is off by less than 2.4e-5 at |q| <= 127,
// so only values that close to a tie (about one in 20000), and scales whose reciprocal overflows, take the f64 quotient,
// which never rounds across a tie (x and scale have 24 bits each).
__device__ __forceinline__ int code_of(float x, float scale, float inv) {
  if (!(scale > 0.0f) || scale == INFINITY) return 0;
  const float t = x * inv;
  float q = rintf(t);
  if (!(fabsf(t - q) < 0.49997f)) q = (float)rint((double)x / (double)scale);
  return (int)fminf(fmaxf(q, -127.0f), 127.0f);
}

template <typename T>
__device__ __forceinline__ float4 load4(const T *p);
template <>
__device__ __forceinline__ float4 load4<float>(const float *p) { return __ldcs((const float4 *)p); }
template <>
__device__ __forceinline__ float4 load4<__half>(const __half *p) {
  const uint2 w = __ldcs((const uint2 *)p);
  const float2 a = __half22float2(*(const __half2 *)&w.x), b = __half22float2(*(const __half2 *)&w.y);
  return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ float load1(const float *p) { return *p; }
__device__ __forceinline__ float load1(const __half *p) { return __half2float(*p); }

// One value of a stored block.
__device__ __forceinline__ float stored(const uint8_t *blk, int which, int pos, int ch, int HDP) {
  int lane, wi, e;
  if (which == 0) {
    const int KS = HDP >> 4;
    lane = ((pos >> 3) * 2 + (pos & 1)) * 4 + ((ch & 15) >> 2), wi = ((pos & 7) >> 1) * KS + (ch >> 4), e = ch & 3;
  } else {
    lane = (ch & 7) * 4 + (pos >> 3), wi = (ch >> 3) * 2 + ((pos & 7) >> 2), e = pos & 3;
  }
  const uint32_t w = *(const uint32_t *)(blk + (size_t)which * kBlock * HDP + (wi >> 2) * 512 + lane * 16 + (wi & 3) * 4);
  return kv8::unpack(w, e) * ((const float *)(blk + (size_t)2 * kBlock * HDP))[which];
}

// One (stream, head, keys or values): the thread block of x == 0 takes the first and the last block that the rows touch, one
// after the other, since the first may need the tail that the last one replaces; the others take one block in between.
//
// Bound by HBM: 4 bytes in, 1 out.  The rows are staged in shared memory so that both the reads (rows) and the writes (the
// fragment order, 16 bytes a lane) are whole sectors; 8 to 16 thread blocks an SM keep 8 KB of loads each in flight.
template <typename T>
__global__ void __launch_bounds__(kThreads) k_kv8_write(const WriteParams p) {
  extern __shared__ float sx[];  // [32][HDP + pad]
  __shared__ float wmax[kThreads / 32];
  fa_grid_dep_sync();
  const int h = blockIdx.y >> 1, which = blockIdx.y & 1, s = blockIdx.z;
  int start, count;
  bool bad;
  p.rows.of(s, start, count, bad);
  if (bad && blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) atomicOr(p.status + 3, kStatusKv8Length);
  if (count <= 0) return;
  const int end = start + count, first = start / kBlock, last = (end - 1) / kBlock;
  const int HD = p.HD, HDP = p.HDP, pitch = HDP + 1;  // odd: the values' order reads columns
  const size_t unit = (size_t)s * p.H + h;
  float *tail = p.tail + (unit * 2 + which) * kBlock * HD;
  const T *src = (const T *)p.src[which] + ((size_t)s * p.rows.T - start) * p.ld + (size_t)h * HD;  // + position * ld
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int turns = blockIdx.x == 0 ? 1 + (last > first) : (int)blockIdx.x < last - first;
  for (int turn = 0; turn < turns; turn++) {
    const int b = blockIdx.x == 0 ? (turn ? last : first) : first + (int)blockIdx.x, base = b * kBlock;
    uint8_t *blk = p.codes + (unit * p.nblk + b) * kv8::block_bytes(HDP);
    const int held = max(0, start - base);              // rows of this block from before the call
    const int rows = min(kBlock, end - base);
    const bool kept = held > 0 && p.tag[unit * 2 + which] == b;  // (read before the barrier in front of its update)
    float top = 0.0f;
    bool nan = false;
    auto put = [&](int r, int d, float x) {
      sx[r * pitch + d] = x;
      top = fmaxf(top, fabsf(x));
      nan |= x != x;
    };
    if (p.vec) {
      const int n4 = HDP / 4;
      for (int i = threadIdx.x; i < kBlock * n4; i += kThreads) {
        const int r = i / n4, d = (i - r * n4) * 4;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < rows && d < HD) {
          if (r >= held) x = load4(src + (size_t)(base + r) * p.ld + d);
          else if (kept) x = *(const float4 *)(tail + r * HD + d);
          else x = make_float4(stored(blk, which, r, d, HDP), stored(blk, which, r, d + 1, HDP), stored(blk, which, r, d + 2, HDP), stored(blk, which, r, d + 3, HDP));
        }
        put(r, d, x.x), put(r, d + 1, x.y), put(r, d + 2, x.z), put(r, d + 3, x.w);
      }
    } else {
      for (int i = threadIdx.x; i < kBlock * HDP; i += kThreads) {
        const int r = i / HDP, d = i - r * HDP;
        float x = 0.0f;
        if (r < rows && d < HD) x = r >= held ? load1(src + (size_t)(base + r) * p.ld + d) : kept ? tail[r * HD + d] : stored(blk, which, r, d, HDP);
        put(r, d, x);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0) wmax[warp] = top;
    const bool any_nan = __syncthreads_or(nan);
    top = fmaxf(fmaxf(wmax[0], wmax[1]), fmaxf(wmax[2], wmax[3]));
    const float scale = any_nan ? __int_as_float(0x7fc00000) : top / 127.0f, inv = 1.0f / scale;
    const int words = HDP / 4, KS = HDP / 16;
    for (int i = threadIdx.x; i < words * 8; i += kThreads) {  // 16 bytes: words 4c .. 4c+3 of a lane
      const int ln = i & 31, c = i >> 5;
      uint32_t w[4];
#pragma unroll
      for (int u = 0; u < 4; u++) {
        int pos, ch, q[4];
        if (which == 0) {
          kv8::k_place(4 * c + u, ln, KS, pos, ch);
#pragma unroll
          for (int e = 0; e < 4; e++) q[e] = code_of(sx[pos * pitch + ch + e], scale, inv);
        } else {
          kv8::v_place(4 * c + u, ln, pos, ch);
#pragma unroll
          for (int e = 0; e < 4; e++) q[e] = code_of(sx[(pos + e) * pitch + ch], scale, inv);
        }
        w[u] = kv8::pack4(q);
      }
      *(uint4 *)(blk + (size_t)which * kBlock * HDP + (size_t)c * 512 + ln * 16) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    if (threadIdx.x == 0) ((float *)(blk + (size_t)2 * kBlock * HDP))[which] = scale;
    if (b == last) {  // its f32 rows stay: a row that joins the block codes it anew
      for (int i = threadIdx.x; i < rows * HD; i += kThreads) {
        const int r = i / HD, d = i - r * HD;
        if (r >= held || !kept) tail[i] = sx[r * pitch + d];
      }
      if (threadIdx.x == 0) p.tag[unit * 2 + which] = b;
    }
    __syncthreads();
  }
}

struct ReadParams {
  const uint8_t *codes;
  float *out[2];
  int row0, rows, H, HD, HDP, nblk;
};

__global__ void __launch_bounds__(kThreads) k_kv8_read(const ReadParams p) {
  extern __shared__ __align__(16) uint8_t sb[];  // half a block
  fa_grid_dep_sync();
  const int h = blockIdx.y >> 1, which = blockIdx.y & 1, s = blockIdx.z, HD = p.HD, HDP = p.HDP;
  const int b = p.row0 / kBlock + blockIdx.x, half = kBlock * HDP;
  const uint8_t *blk = p.codes + (((size_t)s * p.H + h) * p.nblk + b) * kv8::block_bytes(HDP);
  for (int i = threadIdx.x; i < half / 16; i += kThreads) ((uint4 *)sb)[i] = ((const uint4 *)(blk + (size_t)which * half))[i];
  const float scale = ((const float *)(blk + (size_t)2 * half))[which];
  __syncthreads();
  const int KS = HDP >> 4, lo = max(p.row0 - b * kBlock, 0), hi = min(kBlock, p.row0 + p.rows - b * kBlock);
  float *out = p.out[which] + ((size_t)s * p.rows + (size_t)b * kBlock - p.row0) * p.H * HD + (size_t)h * HD;
  for (int i = threadIdx.x; i < (hi - lo) * HD; i += kThreads) {
    const int r = lo + i / HD, d = i % HD;
    int lane, wi, e;
    if (which == 0) lane = ((r >> 3) * 2 + (r & 1)) * 4 + ((d & 15) >> 2), wi = ((r & 7) >> 1) * KS + (d >> 4), e = d & 3;
    else lane = (d & 7) * 4 + (r >> 3), wi = (d >> 3) * 2 + ((r & 7) >> 2), e = r & 3;
    out[(size_t)r * p.H * HD + d] = kv8::unpack(*(const uint32_t *)(sb + (wi >> 2) * 512 + lane * 16 + (wi & 3) * 4), e) * scale;
  }
}

}  // namespace

bool fa_valid_kv8(fa_ctx *ctx, const fa_kv8 *c) { return c && ctx->kv8s.count(const_cast<fa_kv8 *>(c)); }

extern "C" int fa_kv8_create(fa_ctx *ctx, int S, int positions, int H, int HD, fa_kv8 **out) {
  if (!ctx || !out) return fa_fail(ctx, FA_ERR_INVALID, "kvCache8: NULL argument");
  *out = nullptr;
  FA_REQUIRE(ctx, S >= 1 && S <= 65535 && positions >= 1 && positions <= (1 << 24) && H >= 1 && H <= 32767 && HD >= 1 && HD <= 256,
             "kvCache8: %d streams (1..65535), %d positions (1..2^24), %d heads (1..32767) of %d (1..256)", S, positions, H, HD);
  FA_REQUIRE(ctx, !ctx->capturing, "kvCache8: not allowed while a graph is being recorded");
  FA_CHECK_CUDA(ctx, cudaSetDevice(ctx->device));
  fa_kv8 c;
  c.S = S, c.P = positions, c.H = H, c.HD = HD;
  c.HDP = kv8::stored_width(HD), c.nblk = ceil_div(positions, kBlock);
  const size_t units = (size_t)S * H;
  const size_t codes = units * c.nblk * kv8::block_bytes(c.HDP), tail = units * 2 * kBlock * HD * 4, tag = units * 2 * 4, tickets = units * 4;
  size_t blk = 0;
  int rc = fa_block_acquire(ctx, codes, (void **)&c.codes, &blk);
  if (rc == FA_OK) rc = fa_block_acquire(ctx, tail, (void **)&c.tail, &blk);
  if (rc == FA_OK) rc = fa_block_acquire(ctx, tag, (void **)&c.tag, &blk);
  if (rc == FA_OK) rc = fa_block_acquire(ctx, tickets, (void **)&c.tickets, &blk);
  // zero codes with zero scales: a position that nothing was written to reads as zeros; no tail holds a block yet
  if (rc == FA_OK && (cudaMemsetAsync(c.codes, 0, codes, ctx->stream) != cudaSuccess || cudaMemsetAsync(c.tag, 0xff, tag, ctx->stream) != cudaSuccess ||
                      cudaMemsetAsync(c.tickets, 0, tickets, ctx->stream) != cudaSuccess))
    rc = fa_fail(ctx, FA_ERR_CUDA, "kvCache8: %s", cudaGetErrorString(cudaGetLastError()));
  if (rc != FA_OK) {
    for (void *q : {(void *)c.codes, (void *)c.tail, (void *)c.tag, (void *)c.tickets})
      if (q) fa_block_release(ctx, q);
    return rc;
  }
  *out = new fa_kv8(c);
  ctx->kv8s.insert(*out);
  return FA_OK;
}

extern "C" int fa_kv8_free(fa_ctx *ctx, fa_kv8 *c) {
  if (!ctx) return fa_fail(ctx, FA_ERR_INVALID, "freeKvCache8: NULL context");
  if (!c) return FA_OK;
  FA_REQUIRE(ctx, fa_valid_kv8(ctx, c), "freeKvCache8: unknown or already freed handle");
  fa_block_release(ctx, c->codes);
  fa_block_release(ctx, c->tail);
  fa_block_release(ctx, c->tag);
  fa_block_release(ctx, c->tickets);
  ctx->kv8s.erase(c);
  delete c;
  return FA_OK;
}

// Rows [S*T] of keys and of values, with a row pitch of ld elements, into the cache.
int fa_kv8_write_rows(fa_ctx *ctx, fa_kv8 *c, const void *k, const void *v, bool f16, long long ld, int T, int n, const float *pos,
                      const float *counts) {
  if (T == 0) return FA_OK;
  WriteParams p{};
  p.src[0] = k, p.src[1] = v, p.ld = ld;
  p.codes = c->codes, p.tail = c->tail, p.tag = c->tag;
  p.rows = kv8::Rows{pos, counts, n, T, c->P};
  p.H = c->H, p.HD = c->HD, p.HDP = c->HDP, p.nblk = c->nblk;
  const uintptr_t mask = f16 ? 7 : 15;
  p.vec = c->HD % 4 == 0 && ld % 4 == 0 && (((uintptr_t)k | (uintptr_t)v) & mask) == 0;
  p.status = ctx->dev_status;
  const int touched = pos ? ceil_div(T + kBlock - 1, kBlock) : (n + T - 1) / kBlock - n / kBlock + 1;
  const dim3 grid(touched > 1 ? touched - 1 : 1, 2 * c->H, c->S);  // (the first thread block takes two)
  const size_t smem = (size_t)kBlock * (c->HDP + 1) * 4;
  {
    LaunchScope ls(ctx, "kv8_write");
    fa_launch_dep(ctx, f16 ? k_kv8_write<__half> : k_kv8_write<float>, grid, dim3(kThreads), smem, p);
  }
  FA_LAUNCH_CHECK(ctx, "kv8_write");
  return FA_OK;
}

// An optional [S] tensor of whole numbers that only the device reads.
int fa_kv8_per_stream(fa_ctx *ctx, const fa_tensor *t, int S, const char *op, const char *what, const float **out) {
  *out = nullptr;
  if (!t) return FA_OK;
  FA_REQUIRE(ctx, fa_valid(ctx, t) && t->storage == FA_F32 && (long long)t->rows * t->cols == S, "%s: %s needs %d f32 values, one per stream", op, what, S);
  FA_TRY(fa_touch_f32(ctx, t));
  *out = (const float *)t->dptr;
  return FA_OK;
}

extern "C" int fa_kv8_write(fa_ctx *ctx, fa_kv8 *c, const fa_tensor *k, const fa_tensor *v, int n, const fa_tensor *pos, const fa_tensor *counts) {
  if (!ctx) return fa_fail(ctx, FA_ERR_INVALID, "kvWrite8: NULL context");
  FA_REQUIRE(ctx, fa_valid_kv8(ctx, c), "kvWrite8: unknown cache handle");
  FA_REQUIRE(ctx, fa_valid(ctx, k) && fa_valid(ctx, v), "kvWrite8: unknown tensor handle");
  FA_CHECK_CUDA(ctx, cudaSetDevice(ctx->device));
  FA_REQUIRE(ctx, k->storage == v->storage, "kvWrite8: keys and values of different storage");
  FA_REQUIRE(ctx, (long long)k->cols == (long long)c->H * c->HD && v->cols == k->cols, "kvWrite8: keys and values need %lld columns", (long long)c->H * c->HD);
  FA_REQUIRE(ctx, k->rows == v->rows && k->rows % c->S == 0, "kvWrite8: %d and %d rows for %d streams", k->rows, v->rows, c->S);
  const int T = k->rows / c->S;
  FA_REQUIRE(ctx, pos ? T <= c->P : n >= 0 && T <= c->P - n, "kvWrite8: rows %d..%d of a cache of %d positions", n, n + T, c->P);
  FA_TRY(fa_touch_f32(ctx, k));
  FA_TRY(fa_touch_f32(ctx, v));
  const float *dp, *dc;
  FA_TRY(fa_kv8_per_stream(ctx, pos, c->S, "kvWrite8", "pos", &dp));
  FA_TRY(fa_kv8_per_stream(ctx, counts, c->S, "kvWrite8", "counts", &dc));
  return fa_kv8_write_rows(ctx, c, k->dptr, v->dptr, k->storage == FA_F16, k->cols, T, n, dp, dc);
}

extern "C" int fa_kv8_read(fa_ctx *ctx, fa_kv8 *c, int row0, int rows, fa_tensor **out_k, fa_tensor **out_v) {
  if (!ctx || !out_k || !out_v) return fa_fail(ctx, FA_ERR_INVALID, "kvRead8: NULL argument");
  *out_k = *out_v = nullptr;
  FA_REQUIRE(ctx, fa_valid_kv8(ctx, c), "kvRead8: unknown cache handle");
  FA_REQUIRE(ctx, row0 >= 0 && rows >= 0 && rows <= c->P - row0, "kvRead8: rows %d..%lld of a cache of %d positions", row0, (long long)row0 + rows, c->P);
  FA_REQUIRE(ctx, (long long)c->S * rows <= 0x7fffffffLL && (long long)c->H * c->HD <= 0x7fffffffLL, "kvRead8: result too large");
  FA_CHECK_CUDA(ctx, cudaSetDevice(ctx->device));
  fa_tensor *k = nullptr, *v = nullptr;
  FA_TRY(fa_tensor_new(ctx, c->S * rows, c->H * c->HD, FA_F32, true, &k));
  int rc = fa_tensor_new(ctx, c->S * rows, c->H * c->HD, FA_F32, true, &v);
  if (rc == FA_OK && rows) {
    ReadParams p{};
    p.codes = c->codes, p.out[0] = (float *)k->dptr, p.out[1] = (float *)v->dptr;
    p.row0 = row0, p.rows = rows, p.H = c->H, p.HD = c->HD, p.HDP = c->HDP, p.nblk = c->nblk;
    const dim3 grid((row0 + rows - 1) / kBlock - row0 / kBlock + 1, 2 * c->H, c->S);
    LaunchScope ls(ctx, "kv8_read");
    const cudaError_t e = fa_launch_dep(ctx, k_kv8_read, grid, dim3(kThreads), (size_t)kBlock * c->HDP, p);
    if (e != cudaSuccess) rc = fa_fail(ctx, FA_ERR_CUDA, "launch kv8_read: %s", cudaGetErrorString(e));
  }
  if (rc != FA_OK) {
    fa_free_tensor(ctx, k);
    if (v) fa_free_tensor(ctx, v);
    return rc;
  }
  *out_k = k, *out_v = v;
  return FA_OK;
}
