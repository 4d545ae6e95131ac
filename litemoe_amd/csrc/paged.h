// The paged KV cache of one layer, and rotary positions of a pair, as the
// kernels of kv_paged.hip, kv_evict.hip and attn_decode_paged.hip see them.
#pragma once

#include "internal.h"

namespace lm {

// k, v [pages, heads, page, D]; position j of a row lies in page
// table[row][j >> shift] at j & (page - 1). An entry outside [0, pages) names no
// page: its positions are neither written nor attended.
struct PagedKV {
  bf16 *k, *v;
  int64_t pages;
  int width;  // entries of a table row
  int shift;  // log2 of the page's positions
  int heads;
};

constexpr int kMinPageShift = 4, kMaxPageShift = 16;

// log2 of a page's positions, or -1: pages hold 16 to 65536, a power of two.
inline int page_shift(int64_t page) {
  for (int s = kMinPageShift; s <= kMaxPageShift; ++s)
    if (page == (int64_t)1 << s) return s;
  return -1;
}

inline bool aligned16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
// Two buffers of `bytes` that are one, or share none.
inline bool in_place_or_apart(const void *x, const void *y, int64_t bytes) {
  const intptr_t a = reinterpret_cast<intptr_t>(x), b = reinterpret_cast<intptr_t>(y);
  return a == b || a + bytes <= b || b + bytes <= a;
}

// cos | sin [table_len, rotary]: the first `rotary` channels of a head are turned
// in pairs (i, i + rotary / 2) (neox) or (2 i, 2 i + 1).
struct Rotation {
  const void *table;
  int64_t table_len;
  int rotary;
  bool f32;   // table type: fp32, or bf16
  bool neox;
};

// One pair. With an fp32 table the sums are fp32, rounded where they are stored, one
// product of each in its sum (said here, so that every kernel rounds the same way);
// with a bf16 table each product and each sum is rounded to bf16, the
// arithmetic of lm_rope_kv_write.
__device__ __forceinline__ void turn_pair(bool f32, float x1, float x2, float c, float s, float &o1, float &o2) {
  if (f32) {
    o1 = __builtin_fmaf(x1, c, -(x2 * s));
    o2 = __builtin_fmaf(x2, c, x1 * s);
  } else {
    o1 = round_bf16(x1 * c) - round_bf16(x2 * s);
    o2 = round_bf16(x2 * c) + round_bf16(x1 * s);
  }
}

// Checks shared by the entry points.
inline int paged_args_ok(int64_t width, int64_t pages, int64_t page, int64_t head_dim) {
  if (width <= 0 || pages <= 0 || pages > INT32_MAX || page <= 0) return LM_EINVAL;
  if (page_shift(page) < 0 || (head_dim != 64 && head_dim != 128)) return LM_EUNSUPPORTED;
  if (width > ((int64_t)1 << 30) / page) return LM_EINVAL;  // positions of a row fit 30 bits
  return LM_OK;
}
inline bool rotation_ok(const void *table, int64_t table_len, int64_t rotary, int64_t head_dim) {
  return table && aligned16(table) && table_len > 0 && rotary > 0 && rotary % 16 == 0 && rotary <= head_dim;
}

}  // namespace lm
