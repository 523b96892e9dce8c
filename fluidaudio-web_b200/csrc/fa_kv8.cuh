// The 8-bit key and value cache: layout and device helpers shared by the kernels that write and read it.
//
// A block holds 32 consecutive positions of one head of one stream: K 32 x HDP codes, V 32 x HDP codes, then the two scales.
// A code is u = q + 128 with q = rint(x / scale) in -127..127 and scale = max|x| / 127 over the rows that the block holds, so
// x is read as (u - 128) * scale: one rounding, half a step of the block's largest value / 127 at most.  0x6400 | u is the f16
// 1024 + u, so two codes become f16 operands u - 128 with a byte permutation and a subtraction.  (Signs and magnitudes would be
// f16 subnormals as they stand, an instruction less a word; but the tensor cores align products by exponent fields, and the
// leading zeros of subnormals cost the sums three bits and more: 3e-6 instead of 3e-7 from float64.)
//
// The codes lie in the order in which the lanes of a warp take them as operands of m16n8k16 products (B fragments: lane
// (g, t) = (lane / 4, lane % 4) holds column g and k = 2t, 2t+1, 2t+8, 2t+9), 16 bytes a lane and 512 a warp:
//   scores   column = position, k = channel: word (j, ks) of a lane is position 8 (g/2) + 2j + g%2, channels 16 ks + 4t ..+3;
//   values   column = channel, k = position: word (i, kk) of a lane is channel 8 i + g, positions 8t + 4 kk ..+3.
// The sum over k may run in any order, so the k slots 2t, 2t+1, 2t+8, 2t+9 simply ARE the four neighbours above; and the
// positions are dealt to the score columns so that a lane's weights after the softmax (columns 2t, 2t+1 of the four j) are
// those of positions 8t..8t+7, which is what it needs as the row operand of the second product: nothing moves between lanes.
#pragma once

#include "fa_internal.cuh"

namespace kv8 {

constexpr int kBlock = 32;

// widths that the attention kernels are built for; a head is stored with the smallest that holds it, zeros behind it
inline int stored_width(int HD) { return HD <= 32 ? 32 : HD <= 64 ? 64 : HD <= 96 ? 96 : HD <= 128 ? 128 : 256; }
__host__ __device__ constexpr size_t block_bytes(int HDP) { return (size_t)2 * kBlock * HDP + 16; }

// code e of a word
__device__ __forceinline__ float unpack(uint32_t w, int e) { return (float)((int)(w >> (8 * e) & 255u) - 128); }

// Where stream s's new rows go: `start` = pos[s] or n, `count` = counts[s] or T rows, both inside the cache.
struct Rows {
  const float *pos, *counts;  // [S] on the device, or NULL
  int n, T, P;
  __device__ __forceinline__ void of(int s, int &start, int &count, bool &bad) const {
    bad = false;
    start = n, count = T;
    if (pos) {
      const float f = pos[s];
      bad |= !(f >= 0.0f && f <= (float)P);
      start = f >= 0.0f ? (int)fminf(f, (float)P) : 0;
    }
    if (counts) {
      const float f = counts[s];
      bad |= !(f >= 0.0f && f <= (float)T);
      count = f >= 0.0f ? (int)fminf(f, (float)T) : 0;
    }
    if (count > P - start) bad = true, count = P - start;
  }
};

}  // namespace kv8

bool fa_valid_kv8(fa_ctx *ctx, const fa_kv8 *c);
// host side, shared by the entry points (fa_kv8.cu)
int fa_kv8_write_rows(fa_ctx *ctx, fa_kv8 *c, const void *k, const void *v, bool f16, long long ld, int T, int n, const float *pos,
                      const float *counts);
int fa_kv8_per_stream(fa_ctx *ctx, const fa_tensor *t, int S, const char *op, const char *what, const float **out);
