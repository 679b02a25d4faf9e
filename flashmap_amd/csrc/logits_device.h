// Rows of logits in bf16, fp16 or float32, read 16 bytes at a time from any alignment.
#pragma once

#include "fm_device.h"

namespace fm {

enum LogitType { LOGITS_BF16 = 0, LOGITS_F16 = 1, LOGITS_F32 = 2 };

// Eight consecutive logits as they are stored (few registers while a tile is in flight).
template <int TY>
struct Chunk {
  static constexpr int WORDS = TY == LOGITS_F32 ? 8 : 4, PER_WORD = 8 / WORDS;
  uint32_t w[WORDS];
  // The compiler takes the words as new from here on: the logits decoded before are not
  // kept for a later pass over them (32 registers, which would spill).
  __device__ __forceinline__ void forget() {
#pragma unroll
    for (int q = 0; q < WORDS; ++q) asm volatile("" : "+v"(w[q]));
  }
  __device__ __forceinline__ float at(int j) const {
    const uint32_t v = w[j / PER_WORD];
    if (TY == LOGITS_F32) return __uint_as_float(v);
    if (TY == LOGITS_BF16) return j & 1 ? bf16_hi(v) : bf16_lo(v);
    return j & 1 ? f16_hi(v) : f16_lo(v);
  }
  // -inf in the place of logit j.
  __device__ __forceinline__ void drop(int j) {
    uint32_t &v = w[j / PER_WORD];
    if (TY == LOGITS_F32)
      v = 0xFF800000u;
    else
      v = j & 1 ? (v & 0xFFFFu) | (TY == LOGITS_BF16 ? 0xFF800000u : 0xFC000000u)
                : (v & 0xFFFF0000u) | (TY == LOGITS_BF16 ? 0xFF80u : 0xFC00u);
  }
};

// A row as 16-byte granules from the one its first logit lies in: `skip` logits of that
// granule come before the row, and the last granule may end past it. Loads are of whole
// granules with a logit of the row in them (no allocation ends inside one); the logits
// around the row are dropped after the load.
template <int TY>
struct RowView {
  static constexpr int ES = TY == LOGITS_F32 ? 4 : 2;
  const char *from;
  uint32_t skip, vocab, last;  // last: the row's last granule
  __device__ __forceinline__ RowView(const char *src, int64_t columns) {
    skip = (uint32_t)((uintptr_t)src & 15) / ES;
    from = src - skip * ES;
    vocab = (uint32_t)columns;
    last = (uint32_t)(((uint64_t)skip + vocab - 1) * ES / 16);
  }
  // Chunk g: the logits of columns 8 g - skip to 8 g - skip + 7.
  __device__ __forceinline__ Chunk<TY> chunk(uint32_t g) const {
    Chunk<TY> c;
#pragma unroll
    for (int h = 0; h < ES / 2; ++h) {
      const uint32_t n = g * (ES / 2) + h;
      const u32x4_t v = load16(from + 16 * (uint64_t)(n < last ? n : last));
#pragma unroll
      for (int q = 0; q < 4; ++q) c.w[4 * h + q] = v[q];
    }
    return c;
  }
  // Whether some of n chunks from g on reach past either end.
  __device__ __forceinline__ bool edge(uint32_t g, uint32_t n) const {
    return (g == 0 && skip != 0) || 8 * ((uint64_t)g + n) > (uint64_t)skip + vocab;
  }
  __device__ __forceinline__ void trim(Chunk<TY> &c, uint32_t g) const {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (8 * g - skip + j >= vocab) c.drop(j);
  }
};

}  // namespace fm
