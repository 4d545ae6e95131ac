// The quantising KV-cache store and the read-back (format: kv_quant.h).
//
// Both move each element once and are bound by memory: 256 bytes of bf16 and 68
// (4 bits) or 132 (8 bits) bytes of cache per (row, KV head). Eight lanes hold a
// 64-channel vector, eight channels each, its key and its value; four of them are
// a block, whose maximum takes two DPP moves. The bf16 side is read and written
// non-temporally, so that the cache's lines stay: 50,688 tokens x 8 heads in 4 bits
// stored in 26.9 us (31.3 without) and read back in 22.1 (25.1): 4.9 and 5.9 TB/s; in
// 8 bits 30.1 and 30.6, 5.4 and 5.1 TB/s. Two or four rows per thread store slower
// (30.9, 30.6). A copy of 1 GiB runs at 4.9 TB/s. Up to some hundred rows both take
// 2.5 us in a graph, 0.9 more than the smallest kernel.
#include "internal.h"
#include "kv_quant.h"

namespace lm {
namespace {

constexpr int kThreads = 256;
constexpr int kLanes = 8;                      // lanes of one vector
constexpr int kRowsPerBlock = kThreads / kLanes;

// Eight bf16 channels to floats: one 16-byte load, or element by element where
// the tensor's strides or address do not allow it.
template <bool kVec>
__device__ __forceinline__ void load8(const bf16 *p, int64_t stride, float *f) {
  if constexpr (kVec) {
    unpack8(__builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(p)), f);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = bf16_to_f32(p[i * stride]);
  }
}

// grid (row tiles, heads): consecutive rows of a head, consecutive positions of a
// prompt, are written as one run of codes and scales. Every load is issued before the
// row's target is known.
template <int kBits, bool kVec>
__global__ void __launch_bounds__(kThreads)
kv_quant_write_kernel(const bf16 *__restrict__ k, int64_t ks0, int64_t ks1, int64_t ks3,
                      const bf16 *__restrict__ v, int64_t vs0, int64_t vs1, int64_t vs3,
                      uint8_t *__restrict__ kc, uint8_t *__restrict__ vc,
                      uint32_t *__restrict__ scales, const int64_t *__restrict__ pos,
                      const uint8_t *__restrict__ active, const int64_t *__restrict__ slots,
                      int64_t rows, int heads, int64_t capacity, int64_t cache_batch) {
  const int64_t row = (int64_t)blockIdx.x * kRowsPerBlock + threadIdx.x / kLanes;
  const int h = blockIdx.y, u = threadIdx.x % kLanes;
  if (row >= rows) return;  // whole groups of eight lanes leave together, here and below
  float kx[8], vx[8];
  load8<kVec>(k + row * ks0 + h * ks1 + 8 * u * ks3, ks3, kx);
  load8<kVec>(v + row * vs0 + h * vs1 + 8 * u * vs3, vs3, vx);
  const int64_t p = pos[row];
  const int64_t slot = slots ? slots[row] : row;
  if (!(active ? active[row] : 1) || p < 0 || p >= capacity || slot < 0 || slot >= cache_batch) return;
  uint32_t kb, vb;
  const Codes8<kBits> kq = quantise8<kBits>(kx, kb), vq = quantise8<kBits>(vx, vb);
  const int64_t at = (slot * heads + h) * capacity + p;
  *reinterpret_cast<Codes8<kBits> *>(kc + at * code_bytes<kBits>() + u * kBits) = kq;
  *reinterpret_cast<Codes8<kBits> *>(vc + at * code_bytes<kBits>() + u * kBits) = vq;
  // lane 0 gathers block 1's bytes from the upper half of its eight lanes (row_half_mirror)
  const uint32_t k1 = (uint32_t)__builtin_amdgcn_mov_dpp((int)kb, 0x141, 0xF, 0xF, true);
  const uint32_t v1 = (uint32_t)__builtin_amdgcn_mov_dpp((int)vb, 0x141, 0xF, 0xF, true);
  if (u == 0) scales[at] = kb | k1 << 8 | vb << 16 | v1 << 24;
}

// What a vector's eight codes stand for, as bf16: the exact product of code and
// scale (denormal results included) in fp32, then bf16, which holds it exactly.
template <int kBits>
__device__ __forceinline__ u32x4 dequantise8(const Codes8<kBits> &c, float s) {
  float f[8];
  unpack8(codes_to_bf16<kBits>(c.w), f);
  u32x4 o;
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = pack_bf16(f[2 * i] * s, f[2 * i + 1] * s);
  return o;
}

template <int kBits>
__global__ void __launch_bounds__(kThreads)
kv_quant_read_kernel(const uint8_t *__restrict__ kc, const uint8_t *__restrict__ vc,
                     const uint32_t *__restrict__ scales, const int64_t *__restrict__ pos,
                     const int64_t *__restrict__ slots, bf16 *__restrict__ k, bf16 *__restrict__ v,
                     int64_t rows, int heads, int64_t capacity, int64_t cache_batch) {
  const int64_t row = (int64_t)blockIdx.x * kRowsPerBlock + threadIdx.x / kLanes;
  const int h = blockIdx.y, u = threadIdx.x % kLanes;
  if (row >= rows) return;
  const int64_t p = pos[row];
  const int64_t slot = slots ? slots[row] : row;
  const bool inside = p >= 0 && p < capacity && slot >= 0 && slot < cache_batch;
  u32x4 ko = {0u, 0u, 0u, 0u}, vo = ko;
  if (inside) {
    const int64_t at = (slot * heads + h) * capacity + p;
    const Codes8<kBits> kq = *reinterpret_cast<const Codes8<kBits> *>(kc + at * code_bytes<kBits>() + u * kBits);
    const Codes8<kBits> vq = *reinterpret_cast<const Codes8<kBits> *>(vc + at * code_bytes<kBits>() + u * kBits);
    const uint32_t w = scales[at];
    ko = dequantise8<kBits>(kq, quant_scale(w, u / 4));
    vo = dequantise8<kBits>(vq, quant_scale(w, 2 + u / 4));
  }
  const int64_t out = ((row * heads + h) * kLanes + u) * 8;
  __builtin_nontemporal_store(ko, reinterpret_cast<u32x4 *>(k + out));
  __builtin_nontemporal_store(vo, reinterpret_cast<u32x4 *>(v + out));
}

bool aligned(const void *p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

// Grid limits: row tiles in x (below 2^32 threads), heads in y.
bool sizes_ok(int64_t rows, int64_t heads, int64_t capacity, int64_t cache_batch) {
  return rows >= 0 && rows <= ((int64_t)1 << 28) && heads > 0 && heads <= 65535 && capacity > 0 && cache_batch > 0;
}

}  // namespace
}  // namespace lm

using namespace lm;

extern "C" int lm_kv_quant_write(const void *k, int64_t ks0, int64_t ks1, int64_t ks3, const void *v,
                                 int64_t vs0, int64_t vs1, int64_t vs3, void *k_codes, void *v_codes,
                                 void *scales, const int64_t *positions, const uint8_t *active,
                                 const int64_t *slots, int64_t rows, int64_t heads, int64_t head_dim,
                                 int64_t capacity, int64_t cache_batch, int64_t bits, void *stream) {
  LM_REQUIRE(sizes_ok(rows, heads, capacity, cache_batch));
  if (head_dim != 64 || (bits != 4 && bits != 8)) return LM_EUNSUPPORTED;
  if (rows == 0) return LM_OK;
  LM_REQUIRE(k && v && k_codes && v_codes && scales && positions);
  LM_REQUIRE(aligned(k, 2) && aligned(v, 2) && aligned(k_codes, 16) && aligned(v_codes, 16) && aligned(scales, 4));
  const bool vec = ks3 == 1 && vs3 == 1 && ks0 % 8 == 0 && ks1 % 8 == 0 && vs0 % 8 == 0 && vs1 % 8 == 0 &&
                   aligned(k, 16) && aligned(v, 16);
  const dim3 grid((unsigned)cdiv(rows, kRowsPerBlock), (unsigned)heads);
  auto kernel = bits == 4 ? (vec ? kv_quant_write_kernel<4, true> : kv_quant_write_kernel<4, false>)
                          : (vec ? kv_quant_write_kernel<8, true> : kv_quant_write_kernel<8, false>);
  kernel<<<grid, kThreads, 0, (hipStream_t)stream>>>(
      (const bf16 *)k, ks0, ks1, ks3, (const bf16 *)v, vs0, vs1, vs3, (uint8_t *)k_codes, (uint8_t *)v_codes,
      (uint32_t *)scales, positions, active, slots, rows, (int)heads, capacity, cache_batch);
  LM_CHECK_LAUNCH();
  return LM_OK;
}

extern "C" int lm_kv_quant_read(const void *k_codes, const void *v_codes, const void *scales,
                                const int64_t *positions, const int64_t *slots, int64_t rows,
                                int64_t heads, int64_t head_dim, int64_t capacity, int64_t cache_batch,
                                int64_t bits, void *k, void *v, void *stream) {
  LM_REQUIRE(sizes_ok(rows, heads, capacity, cache_batch));
  if (head_dim != 64 || (bits != 4 && bits != 8)) return LM_EUNSUPPORTED;
  if (rows == 0) return LM_OK;
  LM_REQUIRE(k_codes && v_codes && scales && positions && k && v);
  LM_REQUIRE(aligned(k_codes, 16) && aligned(v_codes, 16) && aligned(scales, 4) && aligned(k, 16) && aligned(v, 16));
  const dim3 grid((unsigned)cdiv(rows, kRowsPerBlock), (unsigned)heads);
  auto kernel = bits == 4 ? kv_quant_read_kernel<4> : kv_quant_read_kernel<8>;
  kernel<<<grid, kThreads, 0, (hipStream_t)stream>>>(
      (const uint8_t *)k_codes, (const uint8_t *)v_codes, (const uint32_t *)scales, positions, slots, (bf16 *)k,
      (bf16 *)v, rows, (int)heads, capacity, cache_batch);
  LM_CHECK_LAUNCH();
  return LM_OK;
}
