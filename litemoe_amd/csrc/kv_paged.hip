// The paged cache's store, with rotary positions or without, and its read-back.
//
// Work is cut into items of 16-byte units (8 channels). Half layout: an item is
// the unit pair (8u.., rotary/2 + 8u..) of a q or k head; interleaved: one unit,
// four pairs. Channels past `rotary` and v are copied, an item a unit. Items of a
// token are numbered q heads, k heads, v heads; thread i of the grid takes item
// i % items of token i / items. So lanes next to each other read and write 16 bytes next
// to each other, whatever the strides and pages.
//
// Bound by the copy: 50,688 tokens of 24 + 8 + 8 heads of 64 channels (585 MB in and out)
// 110 us, 5.3 TB/s (a copy of 2 GiB 4.9). 64 tokens take 4.0 us, 700 4.7: launch, the
// chain position -> page -> store. Read-back of 64 positions 2.0 us.
//
// The reference keeps one page per row (litemoe/flash_decode.py:10-12) and turns
// whole heads in halves (litemoe/model.py:13-15, 58-67).
#include "paged.h"

namespace lm {
namespace {

constexpr int kThreads = 256;
constexpr int64_t kMaxItems = ((int64_t)1 << 32) - kThreads;  // a grid has fewer than 2^32 threads

struct View {
  const bf16 *p;
  int64_t s0, s1;  // token and head strides
};

struct RotateArgs {
  View q, k, v;
  View q_out, k_out;  // p NULL: not written (written through a cast)
  PagedKV kv;         // k NULL: nothing is stored
  int64_t batch;      // rows of the block table
  Rotation rot;
  int q_heads, kv_heads, dim;
  int rot_items, head_items, v_items;  // of a head: turned items, all items; of a v head
  uint32_t items;                      // of a token
  int64_t total;                       // items of the call
  bool at_i32;
};

// Places in the cache come as int64, or as int32 (a row's `used`).
__device__ __forceinline__ int64_t index_at(const void *p, bool i32, int64_t i) {
  return i32 ? static_cast<const int32_t *>(p)[i] : static_cast<const int64_t *>(p)[i];
}

template <bool kF32>
__device__ __forceinline__ void load_angles(const void *row, int at, float *f) {
  if constexpr (kF32) {
    const f32x4 a = reinterpret_cast<const f32x4 *>(static_cast<const float *>(row) + at)[0];
    const f32x4 b = reinterpret_cast<const f32x4 *>(static_cast<const float *>(row) + at)[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[i] = a[i];
      f[4 + i] = b[i];
    }
  } else {
    unpack8(*reinterpret_cast<const u32x4 *>(static_cast<const bf16 *>(row) + at), f);
  }
}

template <bool kNeox, bool kF32>
__global__ void __launch_bounds__(kThreads)
rotate_write_kernel(RotateArgs a, const int64_t *__restrict__ pos, const void *__restrict__ at,
                    const uint8_t *__restrict__ active, const int64_t *__restrict__ slots,
                    const int32_t *__restrict__ table) {
  const int64_t id = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (id >= a.total) return;
  const int64_t token = (uint64_t)id / a.items;
  int item = (int)(id - token * a.items);
  const bool turned_head = item < (a.q_heads + a.kv_heads) * a.head_items;
  int head, unit;
  if (turned_head) {
    head = item / a.head_items;
    unit = item % a.head_items;
  } else {
    item -= (a.q_heads + a.kv_heads) * a.head_items;
    head = item / a.v_items;
    unit = item % a.v_items;
  }
  const bool is_q = turned_head && head < a.q_heads;
  const View src = is_q ? a.q : turned_head ? a.k : a.v;
  if (turned_head && !is_q) head -= a.q_heads;
  const bf16 *from = src.p + token * src.s0 + head * src.s1;
  // where k and v go
  bf16 *cell = nullptr;
  const int64_t p = pos ? pos[token] : 0;
  if (!is_q && a.kv.k && (!active || active[token])) {
    const int64_t row = slots ? slots[token] : token, j = at ? index_at(at, a.at_i32, token) : p;
    if (row >= 0 && row < a.batch && j >= 0 && (j >> a.kv.shift) < a.kv.width) {
      const int64_t page = table[row * a.kv.width + (j >> a.kv.shift)];
      if (page >= 0 && page < a.kv.pages)
        cell = (turned_head ? a.kv.k : a.kv.v) +
               (((page * a.kv.heads + head) << a.kv.shift) + (j & ((1 << a.kv.shift) - 1))) * a.dim;
    }
  }
  const View dst = is_q ? a.q_out : a.k_out;
  bf16 *back = turned_head && dst.p ? const_cast<bf16 *>(dst.p) + token * dst.s0 + head * dst.s1 : nullptr;
  if (!cell && !back) return;
  auto put = [&](int c, const u32x4 &w) {
    if (back) *reinterpret_cast<u32x4 *>(back + c) = w;
    if (cell) *reinterpret_cast<u32x4 *>(cell + c) = w;
  };
  if (!turned_head || unit >= a.rot_items) {  // copied
    const int c = turned_head ? a.rot.rotary + 8 * (unit - a.rot_items) : 8 * unit;
    put(c, *reinterpret_cast<const u32x4 *>(from + c));
    return;
  }
  const bool in_table = p >= 0 && p < a.rot.table_len;
  const int half = a.rot.rotary / 2;
  const void *row = static_cast<const char *>(a.rot.table) + (in_table ? p : 0) * a.rot.rotary * (kF32 ? 4 : 2);
  if constexpr (kNeox) {
    const u32x4 w1 = *reinterpret_cast<const u32x4 *>(from + 8 * unit);
    const u32x4 w2 = *reinterpret_cast<const u32x4 *>(from + half + 8 * unit);
    float c[8], s[8], x1[8], x2[8], o1[8], o2[8];
    load_angles<kF32>(row, 8 * unit, c);
    load_angles<kF32>(row, half + 8 * unit, s);
    unpack8(w1, x1);
    unpack8(w2, x2);
    u32x4 r1 = w1, r2 = w2;
    if (in_table) {
#pragma unroll
      for (int i = 0; i < 8; ++i) turn_pair(kF32, x1[i], x2[i], c[i], s[i], o1[i], o2[i]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        r1[i] = pack_bf16(o1[2 * i], o1[2 * i + 1]);
        r2[i] = pack_bf16(o2[2 * i], o2[2 * i + 1]);
      }
    }
    put(8 * unit, r1);
    put(half + 8 * unit, r2);
  } else {
    const u32x4 w = *reinterpret_cast<const u32x4 *>(from + 8 * unit);
    u32x4 r = w;
    float c[4], s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (kF32) {
        c[i] = static_cast<const float *>(row)[4 * unit + i];
        s[i] = static_cast<const float *>(row)[half + 4 * unit + i];
      } else {
        c[i] = bf16_to_f32(static_cast<const bf16 *>(row)[4 * unit + i]);
        s[i] = bf16_to_f32(static_cast<const bf16 *>(row)[half + 4 * unit + i]);
      }
    }
    if (in_table) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float o1, o2;
        turn_pair(kF32, lo_f32(w[i]), hi_f32(w[i]), c[i], s[i], o1, o2);
        r[i] = pack_bf16(o1, o2);
      }
    }
    put(8 * unit, r);
  }
}

// A thread a 16-byte unit of k and of v.
__global__ void __launch_bounds__(kThreads)
read_kernel(PagedKV kv, const int32_t *__restrict__ table, int64_t batch, const void *__restrict__ pos, bool pos_i32,
            const int64_t *__restrict__ slots, int dim, int64_t total, bf16 *__restrict__ k, bf16 *__restrict__ v) {
  const int64_t id = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (id >= total) return;
  const uint32_t units = dim / 8, each = kv.heads * units;
  const int64_t token = (uint64_t)id / each;
  const uint32_t item = (uint32_t)(id - token * each);
  const int head = item / units, unit = item % units;
  const int64_t row = slots ? slots[token] : token, j = index_at(pos, pos_i32, token);
  u32x4 wk{0, 0, 0, 0}, wv{0, 0, 0, 0};
  if (row >= 0 && row < batch && j >= 0 && (j >> kv.shift) < kv.width) {
    const int64_t page = table[row * kv.width + (j >> kv.shift)];
    if (page >= 0 && page < kv.pages) {
      const int64_t cell = (((page * kv.heads + head) << kv.shift) + (j & ((1 << kv.shift) - 1))) * dim + 8 * unit;
      wk = *reinterpret_cast<const u32x4 *>(kv.k + cell);
      wv = *reinterpret_cast<const u32x4 *>(kv.v + cell);
    }
  }
  reinterpret_cast<u32x4 *>(k)[id] = wk;
  reinterpret_cast<u32x4 *>(v)[id] = wv;
}

bool view_ok(const void *p, int64_t s0, int64_t s1) { return aligned16(p) && s0 % 8 == 0 && s1 % 8 == 0; }

}  // namespace
}  // namespace lm

using namespace lm;

extern "C" int lm_paged_rotate_write(const lm_paged_rotate_args *args, void *stream) {
  LM_REQUIRE(args);
  const auto &[q, qs0, qs1, k, ks0, ks1, v, vs0, vs1, cos_sin, table_len, rotary, table_f32, neox, positions, at, at_i32,
               active, slots, q_out, qo0, qo1, k_out, ko0, ko1, k_pages, v_pages, block_table, batch, width, pages, page,
               rows, q_heads, kv_heads, head_dim] = *args;
  LM_REQUIRE(rows >= 0 && q_heads >= 0 && kv_heads >= 0 && q_heads + kv_heads > 0 && q_heads <= 65535 &&
             kv_heads <= 65535 && head_dim > 0);
  if (head_dim % 16 || head_dim > 256) return LM_EUNSUPPORTED;
  const bool store = k_pages != nullptr;
  LM_REQUIRE((k_pages == nullptr) == (v_pages == nullptr));
  if (store) {
    const int status = paged_args_ok(width, pages, page, head_dim);
    if (status != LM_OK) return status;
    LM_REQUIRE(batch > 0);
  }
  if (rows == 0) return LM_OK;
  if (store) LM_REQUIRE(block_table && aligned16(k_pages) && aligned16(v_pages) && (positions || at));
  LM_REQUIRE(q_heads == 0 || (q && q_out && view_ok(q, qs0, qs1) && view_ok(q_out, qo0, qo1)));
  LM_REQUIRE(kv_heads == 0 || (k && view_ok(k, ks0, ks1) && (k_out || store) && (!k_out || view_ok(k_out, ko0, ko1))));
  LM_REQUIRE(!store || (v && view_ok(v, vs0, vs1)));
  LM_REQUIRE(cos_sin ? positions && rotation_ok(cos_sin, table_len, rotary, head_dim) : rotary == 0);
  RotateArgs a;
  a.at_i32 = at_i32 != 0;
  a.q = {(const bf16 *)q, qs0, qs1};
  a.k = {(const bf16 *)k, ks0, ks1};
  a.v = {(const bf16 *)v, vs0, vs1};
  a.q_out = {(const bf16 *)q_out, qo0, qo1};
  a.k_out = {(const bf16 *)k_out, ko0, ko1};
  a.kv = {(bf16 *)k_pages, (bf16 *)v_pages, pages, (int)width, store ? page_shift(page) : 0, (int)kv_heads};
  a.batch = batch;
  a.rot = {cos_sin, table_len, (int)rotary, table_f32 != 0, neox != 0};
  a.q_heads = (int)q_heads;
  a.kv_heads = (int)kv_heads;
  a.dim = (int)head_dim;
  a.rot_items = (int)(neox ? rotary / 16 : rotary / 8);
  a.head_items = a.rot_items + (int)(head_dim - rotary) / 8;
  a.v_items = (int)head_dim / 8;
  a.items = (uint32_t)((q_heads + kv_heads) * a.head_items + (store ? kv_heads * a.v_items : 0));
  LM_REQUIRE(rows <= kMaxItems / a.items);
  a.total = rows * a.items;
  auto kernel = neox ? (table_f32 ? rotate_write_kernel<true, true> : rotate_write_kernel<true, false>)
                     : (table_f32 ? rotate_write_kernel<false, true> : rotate_write_kernel<false, false>);
  kernel<<<dim3((unsigned)cdiv(a.total, kThreads)), kThreads, 0, (hipStream_t)stream>>>(a, positions, at, active,
                                                                                        slots, block_table);
  LM_CHECK_LAUNCH();
  return LM_OK;
}

extern "C" int lm_paged_read(const lm_paged_read_args *args, void *stream) {
  LM_REQUIRE(args);
  const auto &[k_pages, v_pages, block_table, batch, width, pages, page, positions, positions_i32, slots, rows, heads,
               head_dim, k, v] = *args;
  LM_REQUIRE(rows >= 0 && batch > 0 && heads > 0 && heads <= 65535);
  const int status = paged_args_ok(width, pages, page, head_dim);
  if (status != LM_OK) return status;
  if (rows == 0) return LM_OK;
  LM_REQUIRE(k_pages && v_pages && block_table && positions && k && v);
  LM_REQUIRE(aligned16(k_pages) && aligned16(v_pages) && aligned16(k) && aligned16(v));
  LM_REQUIRE(rows <= kMaxItems / (heads * head_dim / 8));
  const PagedKV kv{(bf16 *)const_cast<void *>(k_pages), (bf16 *)const_cast<void *>(v_pages), pages, (int)width,
                   page_shift(page), (int)heads};
  const int64_t total = rows * heads * (head_dim / 8);
  read_kernel<<<dim3((unsigned)cdiv(total, kThreads)), kThreads, 0, (hipStream_t)stream>>>(
      kv, block_table, batch, positions, positions_i32 != 0, slots, (int)head_dim, total, (bf16 *)k, (bf16 *)v);
  LM_CHECK_LAUNCH();
  return LM_OK;
}
