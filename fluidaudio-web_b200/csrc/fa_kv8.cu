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
  const void *keys, *values;  // row (s, i) of head h at + (s*T + i)*ld + h*HD
  long long ld;
  uint8_t *codes;
  float *tail;
  int *tag;
  kv8::Rows rows;
  int H, HD, nblk;
  int run;  // blocks of a thread block
  int vec;  // rows may be read four values at a time
  int *status;
};

// One value of a stored block.
__device__ __noinline__ float stored(const uint8_t *blk, int which, int pos, int ch, int HDP) {
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

// Four neighbouring values of a row, zeros from HD on.
__device__ __forceinline__ float4 load4(const float *p) { return __ldcs((const float4 *)p); }
__device__ __forceinline__ float4 load4(const __half *p) {
  const uint2 w = __ldcs((const uint2 *)p);
  const float2 a = __half22float2(*(const __half2 *)&w.x), b = __half22float2(*(const __half2 *)&w.y);
  return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ float load1(const float *p) { return *p; }
__device__ __forceinline__ float load1(const __half *p) { return __half2float(*p); }

__device__ __noinline__ uint32_t exact_code(float x, float scale) {
  return scale > 0.0f && scale < INFINITY ? (uint32_t)(128 + (int)fmin(fmax(rint((double)x / (double)scale), -127.0), 127.0)) : 128u;
}

// The word of four values.  The quotient's integer is taken from the product with 1 / scale, off by less than 2.4e-5 at most
// 127.  Only a word with a value that close to a tie looks closer: the sign of x - h * scale, h the half-integer next to the
// quotient, is that of one fused multiply-add, since rounding keeps signs (h has 8 bits, nothing underflows from 1e-30 on).
// Values that were f16 meet ties often: with f64 quotients there, 24 full clips took 187 us (130 now).  Scales whose reciprocal
// overflows or that are no numbers take the f64 quotient, which never rounds across a tie (x and scale have 24 bits each).
__device__ __forceinline__ uint32_t code4(float x0, float x1, float x2, float x3, float scale, float inv) {
  const float x[4] = {x0, x1, x2, x3};
  constexpr float kMagic = 12583040.0f;  // 1.5 * 2^23 + 128: the sum's low byte is the nearest integer + 128, ties to even
  uint32_t u[4];
  float off = 0.0f;
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const float t = x[e] * inv, r = t + kMagic;
    u[e] = __float_as_uint(r);
    off = fmaxf(off, fabsf(t - (r - kMagic)));
  }
  if (!(scale > 1e-30f && scale < INFINITY)) {
#pragma unroll 1
    for (int e = 0; e < 4; e++) {
      const uint32_t q = exact_code(e < 2 ? (e == 0 ? x0 : x1) : (e == 2 ? x2 : x3), scale);
      if (e == 0) u[0] = q;
      if (e == 1) u[1] = q;
      if (e == 2) u[2] = q;
      if (e == 3) u[3] = q;
    }
  } else if (off >= 0.49997f) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const float t = x[e] * inv, r = (t + kMagic) - kMagic, h = r + copysignf(0.5f, t - r), d = fmaf(-h, scale, x[e]);
      const int below = (int)(h - 0.5f);
      u[e] = (uint32_t)(128 + below + (d > 0.0f || (d == 0.0f && (below & 1))));
    }
  }
  return __byte_perm(__byte_perm(u[0], u[1], 0x0040), __byte_perm(u[2], u[3], 0x0040), 0x5410);
}

// One block, keys (WHICH = 0) or values (1): rows to registers, their largest magnitude, codes to shared memory in the block's
// order, from there 16 bytes a thread.  A thread takes four neighbouring channels of a row of keys, since those are one word,
// and four by four values, whose words are four positions of a channel.
template <typename T, int HDP, int WHICH>
__device__ __forceinline__ void write_block(const WriteParams &p, const T *src, float *tail, uint8_t *blk, int *tag, int b, int held, int rows,
                                            bool is_last, uint32_t *sw, uint32_t *smax) {
  constexpr int N4 = HDP / 4, ITEMS = WHICH ? (2 * HDP + kThreads - 1) / kThreads * 4 : HDP / 16;
  const int HD = p.HD;
  // rows of this block that the tail holds; *tag is the position behind its last (read before the barrier in front of its update)
  const int known = held > 0 && (*tag - 1) >> 5 == b ? *tag - b * kBlock : 0;
  float4 x[ITEMS];
  auto at = [&](int k, int &r, int &d) {  // row and channel of the k-th four values
    if (WHICH == 0) {
      const int i = threadIdx.x + k * kThreads;
      r = i / N4, d = (i - r * N4) * 4;
    } else {
      const int i = threadIdx.x + (k >> 2) * kThreads;
      r = i / N4, d = (i - r * N4) * 4;
      r = r * 4 + (k & 3);
    }
  };
  uint32_t top = 0;  // as bits: infinities and NaNs are above all others
  if (held == 0 && rows == kBlock && HD == HDP && p.vec) {  // a whole block
#pragma unroll
    for (int k = 0; k < ITEMS; k++) {
      int r, d;
      at(k, r, d);
      x[k] = r < kBlock ? load4(src + (long long)r * p.ld + d) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  } else {
#pragma unroll
    for (int k = 0; k < ITEMS; k++) {
      int r, d;
      at(k, r, d);
      x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r >= rows || d >= HD) continue;
      if (r >= held) {
        const T *q = src + (long long)r * p.ld + d;
        if (p.vec) {
          x[k] = load4(q);
        } else {
          x[k].x = load1(q);
          if (d + 1 < HD) x[k].y = load1(q + 1);
          if (d + 2 < HD) x[k].z = load1(q + 2);
          if (d + 3 < HD) x[k].w = load1(q + 3);
        }
      } else {  // (asked for before it is known whether the tail is this block's)
        const float *q = tail + r * HD + d;
        if (HD % 4 == 0) {
          x[k] = *(const float4 *)q;
        } else {
          x[k].x = q[0];
          if (d + 1 < HD) x[k].y = q[1];
          if (d + 2 < HD) x[k].z = q[2];
          if (d + 3 < HD) x[k].w = q[3];
        }
      }
    }
  }
  if (held > known) {  // back in an earlier block: its stored values; past rows that nothing wrote: zeros
#pragma unroll
    for (int k = 0; k < ITEMS; k++) {
      int r, d;
      at(k, r, d);
      if (r < known || r >= held || d >= HD) continue;
      x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (known > 0) continue;
      x[k].x = stored(blk, WHICH, r, d, HDP);
      if (d + 1 < HD) x[k].y = stored(blk, WHICH, r, d + 1, HDP);
      if (d + 2 < HD) x[k].z = stored(blk, WHICH, r, d + 2, HDP);
      if (d + 3 < HD) x[k].w = stored(blk, WHICH, r, d + 3, HDP);
    }
  }
#pragma unroll
  for (int k = 0; k < ITEMS; k++)
    top = max(max(top, max(__float_as_uint(x[k].x) & 0x7fffffffu, __float_as_uint(x[k].y) & 0x7fffffffu)),
              max(__float_as_uint(x[k].z) & 0x7fffffffu, __float_as_uint(x[k].w) & 0x7fffffffu));
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) smax[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 32; w++) top = max(top, smax[w]);
  const float scale = __uint_as_float(top) / 127.0f, inv = 1.0f / scale;
  if (WHICH == 0) {
#pragma unroll
    for (int k = 0; k < ITEMS; k++) {
      int r, d;
      at(k, r, d);
      const int lane = ((r >> 3) * 2 + (r & 1)) * 4 + ((d & 15) >> 2), wi = ((r & 7) >> 1) * (HDP / 16) + (d >> 4);
      sw[(wi >> 2) * 128 + lane * 4 + (wi & 3)] = code4(x[k].x, x[k].y, x[k].z, x[k].w, scale, inv);
    }
  } else {
#pragma unroll
    for (int k = 0; k < ITEMS; k += 4) {
      int r, d;
      at(k, r, d);
      if (r >= kBlock) break;
      uint32_t *w = sw + (d >> 4) * 128 + ((d & 7) * 4 + (r >> 3)) * 4 + (d >> 3 & 1) * 2 + ((r & 7) >> 2);  // channel d's; the next 16 on
      w[0] = code4(x[k].x, x[k + 1].x, x[k + 2].x, x[k + 3].x, scale, inv);
      w[16] = code4(x[k].y, x[k + 1].y, x[k + 2].y, x[k + 3].y, scale, inv);
      w[32] = code4(x[k].z, x[k + 1].z, x[k + 2].z, x[k + 3].z, scale, inv);
      w[48] = code4(x[k].w, x[k + 1].w, x[k + 2].w, x[k + 3].w, scale, inv);
    }
  }
  if (is_last) {  // its f32 rows stay: a row that joins the block codes it anew
#pragma unroll
    for (int k = 0; k < ITEMS; k++) {
      int r, d;
      at(k, r, d);
      if (r >= rows || r < min(held, known)) continue;
      float *q = tail + r * HD + d;
      if (d >= HD) continue;
      if (HD % 4 == 0) {
        *(float4 *)q = x[k];
      } else {
        q[0] = x[k].x;
        if (d + 1 < HD) q[1] = x[k].y;
        if (d + 2 < HD) q[2] = x[k].z;
        if (d + 3 < HD) q[3] = x[k].w;
      }
    }
    if (threadIdx.x == 0) *tag = b * kBlock + rows;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * HDP; i += kThreads) ((uint4 *)(blk + (size_t)WHICH * kBlock * HDP))[i] = ((const uint4 *)sw)[i];
  if (threadIdx.x == 0) ((float *)(blk + (size_t)2 * kBlock * HDP))[WHICH] = scale;
}

// One (stream, head, keys or values) and a run of blocks.  The thread block of x == 0 takes the last block that the rows touch
// too, behind its own: the first may need the tail that the last one replaces.
// Where rows are many, bound by its own instructions, 32 a value at 2.9 of 4 a clock (a run of four blocks shares what a thread
// block has to find out first), above the floor of HBM, 4 bytes in, 1 out; by the latency of a load and two barriers for one row.
// 24 clips of 1500 positions, 20 heads of 64: f32 112 us = 4.1 TB/s in and out, f16 130; of lengths from 0 to 1500 62 us (81 with
// blocks one by one; then ten thread blocks an SM 79, sixteen 106).
template <typename T, int HDP>
__global__ void __launch_bounds__(kThreads, HDP <= 64 ? 8 : HDP <= 128 ? 5 : 3) k_kv8_write(const WriteParams p) {
  __shared__ __align__(16) uint32_t sw[8 * HDP];
  __shared__ uint32_t smax[kThreads / 32];
  fa_grid_dep_wait();
  fa_grid_dep_launch();  // (after the wait: what follows may then read what lies further back without a wait of its own)
  const int h = blockIdx.y >> 1, which = blockIdx.y & 1, s = blockIdx.z;
  int start, count;
  bool bad;
  p.rows.of(s, start, count, bad);
  if (bad && blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) atomicOr(p.status + 3, kStatusKv8Length);
  if (count <= 0) return;
  const int end = start + count, first = start / kBlock, last = (end - 1) / kBlock;
  const size_t unit = (size_t)s * p.H + h;
  float *tail = p.tail + (unit * 2 + which) * kBlock * p.HD;
  const T *src = (const T *)(which ? p.values : p.keys) + ((long long)s * p.rows.T - start) * p.ld + h * p.HD;  // + position * ld
  const int b0 = first + (int)blockIdx.x * p.run, b1 = min(last, b0 + p.run);  // the last block is the first thread block's
  auto one = [&](int b) {
    const int base = b * kBlock, held = max(0, start - base), rows = min(kBlock, end - base);  // rows from before the call, and in all
    uint8_t *blk = p.codes + (unit * p.nblk + b) * kv8::block_bytes(HDP);
    if (which == 0) write_block<T, HDP, 0>(p, src + (long long)base * p.ld, tail, blk, p.tag + unit * 2, b, held, rows, b == last, sw, smax);
    else write_block<T, HDP, 1>(p, src + (long long)base * p.ld, tail, blk, p.tag + unit * 2 + 1, b, held, rows, b == last, sw, smax);
    __syncthreads();
  };
#pragma unroll 1
  for (int b = b0, left = max(0, b1 - b0) + (blockIdx.x == 0); left > 0; left--, b++) one(left == 1 && blockIdx.x == 0 ? last : b);
}

template <typename T>
cudaError_t launch_write(fa_ctx *ctx, const WriteParams &p, dim3 grid, int HDP) {
  auto kernel = HDP == 32 ? k_kv8_write<T, 32> : HDP == 64 ? k_kv8_write<T, 64> : HDP == 96 ? k_kv8_write<T, 96>
              : HDP == 128 ? k_kv8_write<T, 128> : k_kv8_write<T, 256>;
  return fa_launch_dep(ctx, kernel, grid, dim3(kThreads), 0, p);
}

struct ReadParams {
  const uint8_t *codes;
  float *keys, *values;
  int row0, rows, H, HD, nblk;
};

// A word of codes as four values.
__device__ __forceinline__ float4 values4(uint32_t w, float scale) {
  auto one = [&](uint32_t selector) { return (__uint_as_float(__byte_perm(w, 0x4B000000u, selector)) - 8388736.0f) * scale; };  // 2^23 + u
  return make_float4(one(0x7540), one(0x7541), one(0x7542), one(0x7543));
}

// One half of a block: a thread turns one word of keys, or four words of values, into four values of a row, or of four rows.
// Bound by HBM, 1 byte in, 4 out: 24 clips of 1500 positions in 78 us = 6.0 TB/s.
template <int HDP>
__global__ void __launch_bounds__(kThreads) k_kv8_read(const ReadParams p) {
  constexpr int N4 = HDP / 4;
  fa_grid_dep_sync();
  const int h = blockIdx.y >> 1, which = blockIdx.y & 1, s = blockIdx.z, HD = p.HD;
  const int b = p.row0 / kBlock + blockIdx.x;
  const uint8_t *blk = p.codes + (((size_t)s * p.H + h) * p.nblk + b) * kv8::block_bytes(HDP);
  const uint32_t *words = (const uint32_t *)(blk + (size_t)which * kBlock * HDP);
  const float scale = ((const float *)(blk + (size_t)2 * kBlock * HDP))[which];
  const int lo = p.row0 - b * kBlock, hi = lo + p.rows;  // rows lo..hi-1 of the block are asked for
  const long long ld = (long long)p.H * HD;
  float *out = (which ? p.values : p.keys) + ((long long)s * p.rows + (long long)b * kBlock - p.row0) * ld + h * HD;
  auto put = [&](int r, int d, const float4 &x) {
    if (r < lo || r >= hi || d >= HD) return;
    float *o = out + r * ld + d;
    if (HD % 4 == 0) {
      __stcs((float4 *)o, x);
    } else {
      o[0] = x.x;
      if (d + 1 < HD) o[1] = x.y;
      if (d + 2 < HD) o[2] = x.z;
      if (d + 3 < HD) o[3] = x.w;
    }
  };
  if (which == 0) {
#pragma unroll
    for (int k = 0; k < HDP / 16; k++) {
      const int i = threadIdx.x + k * kThreads, r = i / N4, d = (i - r * N4) * 4;
      const int lane = ((r >> 3) * 2 + (r & 1)) * 4 + ((d & 15) >> 2), wi = ((r & 7) >> 1) * (HDP / 16) + (d >> 4);
      put(r, d, values4(words[(wi >> 2) * 128 + lane * 4 + (wi & 3)], scale));
    }
  } else {
    for (int i = threadIdx.x; i < 2 * HDP; i += kThreads) {
      const int r = i / N4 * 4, d = (i - i / N4 * N4) * 4;
      float4 v[4];
#pragma unroll
      for (int c = 0; c < 4; c++) {
        const int ch = d + c, lane = (ch & 7) * 4 + (r >> 3), wi = (ch >> 3) * 2 + ((r & 7) >> 2);
        v[c] = values4(words[(wi >> 2) * 128 + lane * 4 + (wi & 3)], scale);
      }
      put(r, d, make_float4(v[0].x, v[1].x, v[2].x, v[3].x));
      put(r + 1, d, make_float4(v[0].y, v[1].y, v[2].y, v[3].y));
      put(r + 2, d, make_float4(v[0].z, v[1].z, v[2].z, v[3].z));
      put(r + 3, d, make_float4(v[0].w, v[1].w, v[2].w, v[3].w));
    }
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
  p.keys = k, p.values = v, p.ld = ld;
  p.codes = c->codes, p.tail = c->tail, p.tag = c->tag;
  p.rows = kv8::Rows{pos, counts, n, T, c->P};
  p.H = c->H, p.HD = c->HD, p.nblk = c->nblk;
  const uintptr_t mask = f16 ? 7 : 15;
  p.vec = c->HD % 4 == 0 && ld % 4 == 0 && (((uintptr_t)k | (uintptr_t)v) & mask) == 0;
  p.status = ctx->dev_status;
  const int touched = pos ? ceil_div(T + kBlock - 1, kBlock) : (n + T - 1) / kBlock - n / kBlock + 1;
  // runs of four while there are four thread blocks for each place on the SMs all the same
  p.run = (long long)touched * 2 * c->H * c->S >= 128ll * ctx->sm_count ? 4 : 1;
  const dim3 grid(touched > 1 ? ceil_div(touched - 1, p.run) : 1, 2 * c->H, c->S);
  {
    LaunchScope ls(ctx, "kv8_write");
    if (f16) launch_write<__half>(ctx, p, grid, c->HDP);
    else launch_write<float>(ctx, p, grid, c->HDP);
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
    p.codes = c->codes, p.keys = (float *)k->dptr, p.values = (float *)v->dptr;
    p.row0 = row0, p.rows = rows, p.H = c->H, p.HD = c->HD, p.nblk = c->nblk;
    const dim3 grid((row0 + rows - 1) / kBlock - row0 / kBlock + 1, 2 * c->H, c->S);
    LaunchScope ls(ctx, "kv8_read");
    auto kernel = c->HDP == 32 ? k_kv8_read<32> : c->HDP == 64 ? k_kv8_read<64> : c->HDP == 96 ? k_kv8_read<96>
                : c->HDP == 128 ? k_kv8_read<128> : k_kv8_read<256>;
    const cudaError_t e = fa_launch_dep(ctx, kernel, grid, dim3(kThreads), 0, p);
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
