// Split-K decode attention over the quantised KV cache (format: kv_quant.h):
//   out[b, h] = softmax_j(scale q_h . K_j) V,  j < used[b],
// K and V what their codes and scales stand for, on the matrix cores.
//
// A cache position of one KV head takes 68 bytes (4 bits) or 132 (8) instead of
// bf16's 256, so the KV stream that bounds the bf16 kernel is 3.8 or 1.9 times
// shorter, and with the products on vector units (about 35 SIMD cycles per
// position there, against 33 that the 4-bit stream leaves) they would bound it.
//
// Workgroup (kv head, split, row), four or eight waves; a wave takes 64 consecutive
// positions (a stage) at a time, the workgroup's stages in turn.
// Stages pass through LDS: codes and scale words are copied there directly
// (global_load_lds), the next stage while one is computed, each wave its own, no barriers.
//
// Scores: K . q with v_mfma_f32_16x16x32_bf16, A the codes of 16 positions as bf16
// without their scales (exact), one product per block of 32 channels,
//   s_j = sl2 * (2^e0 (c_j0 . q_0) + 2^e1 (c_j1 . q_1)).
// The 8-bit matrix instructions would take the codes unconverted and q in two 8-bit
// parts, but they sum products of unequal size with 2^-14 of the largest lost
// (measured on random operands), where this sums in fp32.
// The G query heads of a KV head fill P = 4, 8 or 16 of the 16 columns; the
// other columns take other positions: column c holds query head c % P of tile
// c / P of a pass, and the B operand is zero where a tile is not its column's, so
// one accumulator holds 16/P tiles and each lane four scores, and no exponential
// is spent on an empty column (G = P).
// Codes stay apart from scales so that a block that stands for NaN, stored with
// codes 0, cannot reach another position's row or column through a product.
//
// P.V: V^T . p with v_mfma_f32_16x16x32_bf16, A the transposed codes as bf16
// (ds_read_b64_tr_b4 / _tr_b8 straight from the stage), B the probabilities times
// 2^e of V's block, the probabilities rounded to bf16 as the bf16 kernel rounds
// them. A lane's scores are four consecutive positions of its column's tile, which is
// the order that B takes them in; tiles 1 to 3 of a pass come to the columns of tile 0
// by row rotation, and only those columns of the result are kept. A query head's
// columns share their running maximum; the waves merge once, at the end.
//
// Reference semantics: litemoe/flash_decode.py:16-22; masking litemoe/cache.py:42-47.
#include "internal.h"
#include "kv_quant.h"

#include <type_traits>

namespace lm {
namespace {

constexpr int kD = 64;
constexpr int kStageKeys = 64;
constexpr int kMaxQkvSplits = 8;
constexpr int64_t kCUs = 256;

// Running maximum before any position: finite, so exp2(kEmpty - m) and
// exp2(-inf - kEmpty) are 0 and the loop needs no special case, and below every
// other finite score.
constexpr float kEmpty = -3.402823466e38f;
// A column's reference lies this much (log2 units) above the score that set it, and
// moves only for a score above it: probabilities are at most 1 and the accumulators are
// seldom rescaled.
constexpr float kAbove = 8.f;
// V's codes enter P.V times 2^-32, which the result takes back. A probability of at most 1
// times a scale of up to 2^125 is finite in bf16, and the products of 2^30 positions with
// the largest values sum to less than 2^127: only a position that stands for NaN makes a
// NaN. At the other end fp32 sums in these units hold 24 bits of values down to 2^-86.
constexpr float kDown = 0x1p-32f, kBack = 0x1p32f;
// K's codes enter the scores times 2^-14, which the scale of the scores takes back: 32
// products of codes up to 448 with q of any size stay finite, as they have to where K's
// scale makes small scores of them.
constexpr float kScoreDown = 0x1p-14f, kScoreBack = 0x1p14f;

template <int kBits>
struct Stage {
  static constexpr int kCode = code_bytes<kBits>();
  static constexpr int kSide = kStageKeys * kCode;        // K codes, then V codes
  static constexpr int kBytes = 2 * kSide + 4 * kStageKeys;  // then the scale words
  static constexpr int kSideCopies = kSide / 1024;
};
// A position's 16-byte chunks are held in the stage in an order of the position's: chunk
// c at c ^ chunk_order(position). The 16 positions of a tile, read 4 (8) bytes by each
// of 64 lanes, then meet every bank once instead of two (four) times, and the
// transposing reads of V meet a bank half as often. Conflict cycles per stage 76 -> 29
// (4 bits), 277 -> 38 (8 bits); in 8 bits 10 rows to 1000 6.9 -> 6.4 us, 128 ragged
// rows 57.2 -> 56.0, in 4 bits no difference.
template <int kBits>
__device__ __forceinline__ int chunk_order(int position) {
  return kBits == 4 ? ((position >> 3) ^ (position >> 4)) & 1 : ((position >> 2) ^ (position >> 3 & 2)) & 3;
}

// Stages of a wave in LDS: one computed, one on its way. Four workgroups of two 4-bit
// stages a wave fit a CU: 128 ragged rows to 4095 positions 35.1 us, with three
// stages 37.7, in 8 bits 59.3 and 62.0; 64 rows to 1279 9.8 and 10.2.
constexpr int kSlots = 2;

// Direct global -> LDS copies (see lds_copy16) of 16 and 4 bytes per lane; kOffset
// moves both addresses. Non-temporal: every byte is read once per step by one
// workgroup, and the whole cache streams through between two reads of it.
template <int kOffset>
__device__ __forceinline__ void stage_copy16(const void *base, uint32_t voff, uint32_t lds) {
  asm volatile("global_load_lds_dwordx4 %0, %1 offset:%2 nt" ::"v"(voff), "s"(base), "n"(kOffset), "{m0}"(lds)
               : "memory");
}
__device__ __forceinline__ void stage_copy4(const void *base, uint32_t voff, uint32_t lds) {
  asm volatile("global_load_lds_dword %0, %1 nt" ::"v"(voff), "s"(base), "{m0}"(lds) : "memory");
}
// Every copy of this wave has arrived; LDS reads are not moved across.
__device__ __forceinline__ void copies_wait() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
// Every LDS access of this wave is done: its bytes may be copied over.
__device__ __forceinline__ void lds_reads_done() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// The value of the lane N places further in its row of 16, round the end (row_ror by 16 - N).
template <int N>
__device__ __forceinline__ uint32_t row_from(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x120 + 16 - N, 0xF, 0xF, false);
}
template <int N>
__device__ __forceinline__ float row_from(float v) {
  return __uint_as_float(row_from<N>(__float_as_uint(v)));
}

// Scale byte kByte of a position's word as a float (quant_scale), in one instruction.
template <int kByte>
__device__ __forceinline__ float scale_of(uint32_t word) {
  float r;
  const uint32_t by = 23;
#define LM_SCALE(sel)                                                                             \
  asm("v_lshlrev_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:" sel \
      : "=v"(r)                                                                                   \
      : "v"(by), "v"(word))
  if constexpr (kByte == 0) LM_SCALE("BYTE_0");
  if constexpr (kByte == 1) LM_SCALE("BYTE_1");
  if constexpr (kByte == 2) LM_SCALE("BYTE_2");
  if constexpr (kByte == 3) LM_SCALE("BYTE_3");
#undef LM_SCALE
  return r;
}

// Reductions over the tiles of a query head: columns c % P equal, one row of 16 lanes.
template <int P>
__device__ __forceinline__ float tiles_max(float v) {
  if constexpr (P <= 8) v = fmaxf(v, row_from<8>(v));
  if constexpr (P <= 4) v = fmaxf(v, row_from<4>(v));
  return v;
}
template <int P>
__device__ __forceinline__ float tiles_sum(float v) {
  if constexpr (P <= 8) v += row_from<8>(v);
  if constexpr (P <= 4) v += row_from<4>(v);
  return v;
}

// Neox rotation of one (x1, x2) pair with the reference's three roundings.
__device__ __forceinline__ void rotate_pair(float x1, float x2, float c, float s, float &o1, float &o2) {
  o1 = round_bf16(round_bf16(x1 * c) - round_bf16(x2 * s));
  o2 = round_bf16(round_bf16(x2 * c) + round_bf16(x1 * s));
}

struct Cache {
  uint8_t *k, *v;     // [batch, kv_heads, capacity, code_bytes]
  uint32_t *scales;   // [batch, kv_heads, capacity]
};

struct Partial {
  float *o;  // [batch, q_heads, splits, 64], times kDown
  float *m;  // [batch, q_heads, splits]
  float *l;  // [batch, q_heads, splits]
};

// Positions of a split of a row of n, in stages, so that ragged rows keep every split
// busy: splits * chunk >= n, splits * inv_splits just above 2^32 (a product in place of a
// division). Cut by the longest row instead, the later splits have only the long rows:
// 20 rows of 4000 to 16000 positions in eight splits 25.2 us against 23.7, 12 rows 17.0
// and 15.9, 8 rows to 32768 23.4 and 20.5; rows of one length are within 2%. A split takes
// `least` positions or more (least_chunk), so a short row leaves its later splits empty.
__device__ __forceinline__ int row_chunk(int n, int splits, uint32_t inv_splits, int least) {
  return max((int)__umulhi((uint32_t)((max(n, 1) - 1) / kStageKeys + splits), inv_splits) * kStageKeys, least);
}

// The fused form's input: see lm_flash_decode_qkv.
struct QkvIn {
  const float *part;      // [splits][batch][(q_heads + 2*kv_heads) * 64], NULL: unfused
  int splits;
  const bf16 *cos_sin;    // [table_len, 64]: cos | sin halves
  int64_t table_len;
  const int64_t *pos;     // [batch] position of the new token
  const uint8_t *active;  // [batch] or NULL (all rows write)
  const int32_t *order;   // [batch] row of workgroup z (longest first), or NULL: row z
};

template <int kBits, int P, bool kFused, int kWaves>
__global__ void __launch_bounds__(kWaves * kWave, 2)
decode_quant_kernel(const bf16 *__restrict__ q, int64_t qs0, int64_t qs1, Cache cache,
                    const int32_t *__restrict__ used, int q_heads, int kv_heads, int64_t capacity,
                    float scale, int max_len, uint32_t inv_splits, int least, int splits, Partial part, QkvIn in,
                    bf16 *__restrict__ out, int out_mb) {
  typedef Stage<kBits> St;
  constexpr int kThreads = kWaves * kWave;
  constexpr int kTiles = 16 / P;   // tiles of 16 positions in one accumulator
  constexpr int kPasses = 4 / kTiles;
  constexpr int kMergeBytes = kWaves * P * (kD + 2) * 4;
  constexpr int kStageBytes = kWaves * kSlots * St::kBytes;
  __shared__ __align__(16) uint8_t smem[kStageBytes > kMergeBytes ? kStageBytes : kMergeBytes];
  // The fused form's row as bf16: rotated q heads, rotated new key, new value.
  __shared__ __align__(16) uint16_t sm_row[kFused ? P + 2 : 1][kD];
  const int split = blockIdx.y, h = blockIdx.x;
  const int64_t b = kFused && in.order ? in.order[blockIdx.z] : blockIdx.z;
  if (kFused && (b < 0 || b >= gridDim.z)) return;  // not a permutation: no row of this call
  const int G = q_heads / kv_heads;
  const int lane = threadIdx.x % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int col = lane % 16, grp = lane / 16;
  const int tile = col / P, head = col % P;   // this column's tile of a pass, its query head

  const int64_t first_pos = ((int64_t)b * kv_heads + h) * capacity;
  uint8_t *const my_stages = smem + wave * kSlots * St::kBytes;
  const uint32_t my_lds = __builtin_amdgcn_readfirstlane(lds_address(my_stages));

  // The fused form's row: 32 / kPairs lanes per head, each kPairs of the rotation's
  // channel pairs (j, 32 + j). These loads are requested first; the row's length, position
  // and mask below are waited for one after the other before the first stage is, and the
  // mask, a byte, with all of these.
  constexpr int kPairs = P / 4, kRowLanes = kD / 2 / kPairs;
  static_assert((P + 2) * kRowLanes <= 4 * kWave, "one pass over the row");
  typedef float pairs_t __attribute__((ext_vector_type(kPairs)));
  const int hs = threadIdx.x / kRowLanes, j0 = (threadIdx.x % kRowLanes) * kPairs;
  const bool row_thread = hs < G + 2;
  pairs_t pa[kMaxQkvSplits], pc[kMaxQkvSplits];
  if constexpr (kFused) {
    if (row_thread) {
      const int64_t ncols = (int64_t)(q_heads + 2 * kv_heads) * kD;
      const int src_head = hs < G ? h * G + hs : (hs == G ? q_heads + h : q_heads + kv_heads + h);
      const float *src = in.part + b * ncols + (int64_t)src_head * kD + j0;
#pragma unroll
      for (int s = 0; s < kMaxQkvSplits; ++s)
        if (s < in.splits) {
          pa[s] = *reinterpret_cast<const pairs_t *>(src + (int64_t)s * gridDim.z * ncols);
          pc[s] = *reinterpret_cast<const pairs_t *>(src + (int64_t)s * gridDim.z * ncols + kD / 2);
        }
    }
  }
  int n = min(used[b], max_len);
  n = (int)min((int64_t)n, capacity);
  const int chunk = splits > 1 ? row_chunk(n, gridDim.y, inv_splits, least) : max_len;
  const int k0 = split * chunk, k1 = min(n, k0 + chunk);
  bool writer = false, own = false;
  int64_t pnew = 0;
  if constexpr (kFused) {
    // The new token is stored by the split whose range holds its position
    // (split 0 when none does); where it is attended too, its codes replace
    // those that the stage was loaded with.
    pnew = in.pos[b];
    const bool writes = (!in.active || in.active[b]) && pnew >= 0 && pnew < capacity;
    const int64_t wsplit = pnew >= 0 && pnew < (int64_t)gridDim.y * chunk ? pnew / chunk : 0;
    writer = writes && split == wsplit;
    own = writer && pnew >= k0 && pnew < k1;
  }
  if (splits > 1 && k0 >= n && !writer) return;  // the combine kernel skips empty splits
  // This wave's stages: stage it starts at position k0 + (it * kWaves + wave) * 64.
  const int left = k1 - k0 - wave * kStageKeys;
  const int niter = left > 0 ? (left + kWaves * kStageKeys - 1) / (kWaves * kStageKeys) : 0;
  // Byte offsets of the lane's chunk in even and odd copies (the order repeats after two).
  constexpr int kChunks = St::kCode / 16;
  uint32_t copy_off[2];
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int position = (c * kWave + lane) / kChunks;
    copy_off[c] = (position - c * kWave / kChunks) * St::kCode + (lane % kChunks ^ chunk_order<kBits>(position)) * 16;
  }
  // Requests stage `it` into its slot, its start a 64-bit scalar. Slots past the range
  // repeat its last position: masked, and never bytes that the row does not hold (an
  // 8-bit code may be a NaN there). So where that position is the new token's, which the
  // cache does not hold yet, they repeat the one before it.
  auto issue = [&](int it, int slot) {
    const int start = k0 + (it * kWaves + wave) * kStageKeys;
    const int last = k1 - 1 - start;
    const int repeat = max(kFused && own && pnew == k1 - 1 ? last - 1 : last, 0);
    const int64_t at = first_pos + start;
    const uint32_t lds = my_lds + slot * St::kBytes;
    const uint8_t *kg = cache.k + at * St::kCode, *vg = cache.v + at * St::kCode;
    // Copy c fills the stage's 1 KB from c * 1024 on, lane l its chunk l.
    if (last >= kStageKeys - 1) {
      stage_copy16<0>(kg, copy_off[0], lds);
      stage_copy16<1024>(kg, copy_off[1], lds);
      if constexpr (kBits == 8) {
        stage_copy16<2 * 1024>(kg, copy_off[0], lds);
        stage_copy16<3 * 1024>(kg, copy_off[1], lds);
      }
      stage_copy16<0>(vg, copy_off[0], lds + St::kSide);
      stage_copy16<1024>(vg, copy_off[1], lds + St::kSide);
      if constexpr (kBits == 8) {
        stage_copy16<2 * 1024>(vg, copy_off[0], lds + St::kSide);
        stage_copy16<3 * 1024>(vg, copy_off[1], lds + St::kSide);
      }
      stage_copy4(cache.scales + at, lane * 4, lds + 2 * St::kSide);
      return;
    }
#pragma unroll
    for (int c = 0; c < St::kSideCopies; ++c) {
      const int position = (c * kWave + lane) / kChunks;
      const uint32_t off = (uint32_t)(position <= last ? position : repeat) * St::kCode + copy_off[c % 2] % St::kCode;
      stage_copy16<0>(kg, off, lds + c * 1024);
      stage_copy16<0>(vg, off, lds + St::kSide + c * 1024);
    }
    stage_copy4(cache.scales + at, (uint32_t)min(lane, last) * 4, lds + 2 * St::kSide);
  };
  if (niter > 0) issue(0, 0);

  if constexpr (kFused) {
    if (row_thread) {
      // Summed over the K slices in ascending order and rounded to bf16 (F.linear's
      // output), then rotated, v as it is.
      const bool rotated = hs <= G && pnew >= 0 && pnew < in.table_len;
      const bf16 *cs = in.cos_sin + (rotated ? pnew : 0) * kD + j0;
      bf16 cw[kPairs], sw[kPairs];
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        cw[i] = cs[i];
        sw[i] = cs[kD / 2 + i];
      }
      pairs_t x1 = pa[0], x2 = pc[0];
#pragma unroll
      for (int s = 1; s < kMaxQkvSplits; ++s)
        if (s < in.splits) {
          x1 += pa[s];
          x2 += pc[s];
        }
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        float o1 = round_bf16(x1[i]), o2 = round_bf16(x2[i]);
        if (rotated) rotate_pair(o1, o2, bf16_to_f32(cw[i]), bf16_to_f32(sw[i]), o1, o2);
        sm_row[hs][j0 + i] = (uint16_t)f32_to_bf16(o1);
        sm_row[hs][kD / 2 + j0 + i] = (uint16_t)f32_to_bf16(o2);
      }
    }
    __syncthreads();
  }
  // The new key (lanes 0-7 of sixteen) and value (8-15), eight channels each, quantised: by
  // the wave that stores them and by the one whose stage holds their position.
  auto quantise_new = [&](uint32_t &byte) {
    float x[8];
    unpack8(*reinterpret_cast<const u32x4 *>(&sm_row[kFused ? G + lane % 16 / 8 : 0][8 * (lane % 8)]), x);
    return quantise8<kBits>(x, byte);
  };
  // Channels 32 bl + 8 grp and on of the column's query head.
  u32x4 qw[2];
  if constexpr (kFused) {
#pragma unroll
    for (int bl = 0; bl < 2; ++bl)
      qw[bl] = *reinterpret_cast<const u32x4 *>(&sm_row[min(head, G)][32 * bl + 8 * grp]);
  } else {
    const bf16 *qp = q + b * qs0 + (int64_t)(h * G + min(head, G - 1)) * qs1 + 8 * grp;
    qw[0] = *reinterpret_cast<const u32x4 *>(qp);
    qw[1] = *reinterpret_cast<const u32x4 *>(qp + 32);
  }
  // B operands of the scores: tile t's are zero outside its columns.
  u32x4 qt[kTiles][2];
#pragma unroll
  for (int t = 0; t < kTiles; ++t)
#pragma unroll
    for (int bl = 0; bl < 2; ++bl)
#pragma unroll
      for (int i = 0; i < 4; ++i) qt[t][bl][i] = tile == t && head < G ? qw[bl][i] : 0u;

  const float sl2 = scale * (1.4426950408889634f * kScoreBack);
  float m = kEmpty, l = 0.f;
  f32x4 acc[4];  // times kDown: channels 16 mm + 4 grp + i of column col, of use where tile is 0
#pragma unroll
  for (int mm = 0; mm < 4; ++mm) acc[mm] = f32x4{0.f, 0.f, 0.f, 0.f};

  // LDS offsets in a stage. K: the lane's bytes of tile 0's block 0 and block 1; a tile
  // further on the order of the blocks' chunks is the other.
  int k_off[2];
#pragma unroll
  for (int bl = 0; bl < 2; ++bl) {
    const int byte8 = bl * (St::kCode / 2) + grp * kBits;
    k_off[bl] = col * St::kCode + (byte8 / 16 ^ chunk_order<kBits>(col)) * 16 + byte8 % 16;
  }
  // V, 4 bits: lane col of a group reads the 16 channels of position 16 (col/4) + 4 grp +
  // col%4 and receives channel col of the group's 16 positions, tiles 0-3 in order. 8
  // bits: lanes 2r and 2r+1 read the 16 channels of position r of the group's eight, four
  // of each tile of a pair; lane col receives channel col of all eight.
  int v_off[kBits / 2];
#pragma unroll
  for (int c = 0; c < kBits / 2; ++c) {
    const int position = kBits == 4 ? 16 * (col / 4) + 4 * grp + col % 4 : 16 * (col / 8) + 4 * grp + col / 2 % 4;
    v_off[c] = St::kSide + position * St::kCode + (c ^ chunk_order<kBits>(position)) * 16 +
               (kBits == 8 ? 8 * (col % 2) : 0);
  }

  auto compute = [&](int it, int slot) {
    uint8_t *st = my_stages + slot * St::kBytes;
    const int start = k0 + (it * kWaves + wave) * kStageKeys;
    const int count = k1 - start;  // positions of the stage that count, if fewer than 64
    if constexpr (kFused) {
      if (own && pnew >= start && pnew < start + kStageKeys) {
        // A stage that holds nothing else repeats the bytes of its position from before,
        // which may be no numbers in 8 bits: every slot takes the new codes.
        const int at = (int)(pnew - start);
        const int until = kBits == 8 && count == 1 ? kStageKeys : at + 1;
        uint32_t byte;
        const Codes8<kBits> c = quantise_new(byte);
        const int side = lane % 16 / 8, byte8 = lane % 8 * kBits;  // of the vector's codes
        for (int to = at + lane / 16; to < until; to += 4)
          *reinterpret_cast<Codes8<kBits> *>(st + side * St::kSide + to * St::kCode +
                                             (byte8 / 16 ^ chunk_order<kBits>(to)) * 16 + byte8 % 16) = c;
        if (lane < 16 && lane % 4 == 0) st[2 * St::kSide + 4 * at + lane / 4] = (uint8_t)byte;
        lds_reads_done();
      }
    }
    // Everything that the stage's products take from LDS is requested before the
    // first product, so that one latency serves them all.
    typedef int i32x2 __attribute__((ext_vector_type(2)));
    typedef __attribute__((address_space(3))) i32x2 lds_i32x2;
    Codes8<kBits> a[4][2];  // tile t: channels 32 bl + 8 grp and on of position 16 t + col
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int bl = 0; bl < 2; ++bl)
        a[t][bl] = *reinterpret_cast<const Codes8<kBits> *>(st + k_off[(t + bl) % 2] + 16 * t * St::kCode);
    u32x4 words[kPasses];  // scale words of the lane's four positions of each pass
#pragma unroll
    for (int p = 0; p < kPasses; ++p)
      words[p] = *reinterpret_cast<const u32x4 *>(st + 2 * St::kSide + 4 * ((p * kTiles + tile) * 16 + 4 * grp));
    i32x2 vt[4][kBits / 4];  // V^T: channel 16 mm + col, eight positions of tiles 2 pr and 2 pr + 1 each
#pragma unroll
    for (int mm = 0; mm < 4; ++mm) {
      if constexpr (kBits == 4) {
        vt[mm][0] = __builtin_amdgcn_ds_read_tr4_b64_v2i32((lds_i32x2 *)(st + v_off[mm / 2] + 8 * (mm % 2)));
      } else {
#pragma unroll
        for (int pr = 0; pr < 2; ++pr)
          vt[mm][pr] = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2 *)(st + v_off[mm] + 32 * pr * St::kCode));
      }
    }
    f32x4 c[kPasses][2];
#pragma unroll
    for (int p = 0; p < kPasses; ++p) c[p][0] = c[p][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int bl = 0; bl < 2; ++bl)
        c[t / kTiles][bl] =
            mfma16x16x32(codes_to_bf16<kBits>(a[t][bl].w, kScoreDown), qt[t % kTiles][bl], c[t / kTiles][bl]);
    float s[kPasses][4];
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        s[p][i] = (c[p][0][i] * scale_of<0>(words[p][i]) + c[p][1][i] * scale_of<1>(words[p][i])) * sl2;
    }
    if (count < kStageKeys) {
      // Masked positions: whatever their bytes hold, score -inf and V's scales 0.
#pragma unroll
      for (int p = 0; p < kPasses; ++p)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool ok = (p * kTiles + tile) * 16 + 4 * grp + i < count;
          words[p][i] = ok ? words[p][i] : 0u;
          s[p][i] = ok ? s[p][i] : -INFINITY;
        }
    }
    float mx = m;
#pragma unroll
    for (int p = 0; p < kPasses; ++p)
#pragma unroll
      for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[p][i]);
    if (__any(mx > m)) {
      mx = fmaxf(mx, xor_lanes<16>(mx));
      mx = tiles_max<P>(fmaxf(mx, xor_lanes<32>(mx)));
      const bool up = mx > m;
      const float to = mx + kAbove;
      const float f = up ? __builtin_amdgcn_exp2f(m - to) : 1.f;
      m = up ? to : m;
      l *= f;
#pragma unroll
      for (int mm = 0; mm < 4; ++mm) acc[mm] *= f;
    }
    // Probabilities rounded to bf16, their sum from the rounded ones (so that a row
    // that one position rules keeps its value: 5 to 15% less error at no cost), times
    // the scale of each block of V, which is exact from 2^-126 up, as bf16 pairs. In two
    // bf16 parts the result would be off by 1.65e-3 (RMS, relative), the output's own
    // rounding, instead of 1.85e-3 to 2.15e-3, for 3 to 9% more time in 4 bits (128 ragged
    // rows 35.0 -> 37.3 us, fused 33.4 -> 39.2, 64 rows to 1279 10.2 -> 10.9) and 1 to 2% in
    // 8; the cache's own rounding is 1.1e-1 and 2.7e-2, so one part is taken, as over a bf16
    // cache.
    uint32_t pb[2][kPasses][2];
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      float e[4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t r = pack_bf16_finite(__builtin_amdgcn_exp2f(s[p][2 * i] - m),
                                            __builtin_amdgcn_exp2f(s[p][2 * i + 1] - m));
        e[2 * i] = lo_f32(r);
        e[2 * i + 1] = hi_f32(r);
        l += e[2 * i];
        l += e[2 * i + 1];
        const uint32_t w0 = words[p][2 * i], w1 = words[p][2 * i + 1];
        pb[0][p][i] = pack_bf16_finite(e[2 * i] * scale_of<2>(w0), e[2 * i + 1] * scale_of<2>(w1));
        pb[1][p][i] = pack_bf16_finite(e[2 * i] * scale_of<3>(w0), e[2 * i + 1] * scale_of<3>(w1));
      }
    }
    // B operands of tiles 2 pr and 2 pr + 1: a pass's first tile from the column's own
    // lanes, the others from the columns that hold them.
    u32x4 bp[2][2];
#pragma unroll
    for (int bl = 0; bl < 2; ++bl)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if constexpr (P == 4) {
          bp[0][bl][i] = pb[bl][0][i];
          bp[0][bl][2 + i] = row_from<4>(pb[bl][0][i]);
          bp[1][bl][i] = row_from<8>(pb[bl][0][i]);
          bp[1][bl][2 + i] = row_from<12>(pb[bl][0][i]);
        } else if constexpr (P == 8) {
#pragma unroll
          for (int pr = 0; pr < 2; ++pr) {
            bp[pr][bl][i] = pb[bl][pr][i];
            bp[pr][bl][2 + i] = row_from<8>(pb[bl][pr][i]);
          }
        } else {
#pragma unroll
          for (int t = 0; t < 4; ++t) bp[t / 2][bl][2 * (t % 2) + i] = pb[bl][t][i];
        }
      }
#pragma unroll
    for (int mm = 0; mm < 4; ++mm)
#pragma unroll
      for (int pr = 0; pr < 2; ++pr) {
        uint32_t w[kBits / 4];
#pragma unroll
        for (int j = 0; j < kBits / 4; ++j) w[j] = (uint32_t)(kBits == 4 ? vt[mm][0][pr] : vt[mm][pr * (kBits / 8)][j]);
        acc[mm] = mfma16x16x32(codes_to_bf16<kBits>(w, kDown), bp[pr][mm / 2], acc[mm]);
      }
  };

  for (int it = 0; it < niter; ++it) {
    copies_wait();  // stage `it` has arrived
    if (it + 1 < niter) {
      lds_reads_done();  // of stage it - 1, whose slot the next one takes
      issue(it + 1, (it + 1) % 2);
    }
    compute(it, it % 2);
  }

  // Stored behind the stream, which does not wait for it.
  if constexpr (kFused) {
    if (writer && wave == 0 && lane < 16) {
      uint32_t byte;
      const Codes8<kBits> c = quantise_new(byte);
      const int64_t at = first_pos + pnew;
      *reinterpret_cast<Codes8<kBits> *>((lane < 8 ? cache.k : cache.v) + at * St::kCode + lane % 8 * kBits) = c;
      if (lane % 4 == 0) reinterpret_cast<uint8_t *>(cache.scales + at)[lane / 4] = (uint8_t)byte;
    }
  }

  // A query head's sum of probabilities: over the four lanes of its columns and the
  // columns of its tiles. The maximum and the accumulators are whole already.
  l += xor_lanes<16>(l);
  l += xor_lanes<32>(l);
  l = tiles_sum<P>(l);
  __syncthreads();  // every wave is done with its stages
  float(*sm_o)[P][kD] = reinterpret_cast<float(*)[P][kD]>(smem);
  float(*sm_m)[P] = reinterpret_cast<float(*)[P]>(smem + kWaves * P * kD * 4);
  float(*sm_l)[P] = sm_m + kWaves;
  if (tile == 0) {
#pragma unroll
    for (int mm = 0; mm < 4; ++mm) *reinterpret_cast<f32x4 *>(&sm_o[wave][head][16 * mm + 4 * grp]) = acc[mm];
    if (grp == 0) {
      sm_m[wave][head] = m;
      sm_l[wave][head] = l;
    }
  }
  __syncthreads();
  for (int t = threadIdx.x; t < G * kD; t += kThreads) {
    const int g = t / kD, c = t % kD;
    float mx = sm_m[0][g];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) mx = fmaxf(mx, sm_m[w][g]);
    float lsum = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float fw = __builtin_amdgcn_exp2f(sm_m[w][g] - mx);
      lsum += sm_l[w][g] * fw;
      o += sm_o[w][g][c] * fw;
    }
    const int hq = h * G + g;
    if (splits == 1) {
      const int64_t at = out_mb ? frag_offset_rows(b, (int64_t)hq * kD + c, out_mb) : (b * q_heads + hq) * kD + c;
      out[at] = (bf16)f32_to_bf16(lsum == 0.f ? 0.f : o / lsum * kBack);
    } else {
      const int64_t at = ((int64_t)b * q_heads + hq) * splits + split;
      part.o[at * kD + c] = o;
      if (c == 0) {
        part.m[at] = mx;
        part.l[at] = lsum;
      }
    }
  }
}

// grid (pairs of query heads, batch), one thread per channel: the splits' partials by
// log-sum-exp, those of kBatch splits requested together (clamped and masked, so that
// none waits behind the row's length). Against batches of 4 or 16 alone and one head
// per workgroup: 3 rows to 4001 positions in 8 splits 7.5 -> 6.7 us, 8 rows to 32768 in 4
// splits 21.7 -> 21.5; four heads per workgroup are slower at 8 splits (7.1).
constexpr int kCombineHeads = 2;
template <int kBatch>
__global__ void __launch_bounds__(kCombineHeads * kD)
decode_quant_combine_kernel(const int32_t *__restrict__ used, int q_heads, int64_t capacity, int max_len,
                            uint32_t inv_splits, int least, int grid_splits, int splits, Partial part,
                            bf16 *__restrict__ out, int out_mb) {
  const int hq = blockIdx.x * kCombineHeads + threadIdx.x / kD;
  if (hq >= q_heads) return;
  const int64_t b = blockIdx.y;
  const int c = threadIdx.x % kD;
  const int64_t base = ((int64_t)b * q_heads + hq) * splits;
  float ms[kBatch], ls[kBatch], os[kBatch];
  auto load = [&](int s0) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int64_t at = base + min(s0 + i, splits - 1);
      ms[i] = part.m[at];
      ls[i] = part.l[at];
      os[i] = part.o[at * kD + c];
    }
  };
  load(0);
  int n = min(used[b], max_len);
  n = (int)min((int64_t)n, capacity);
  const int chunk = row_chunk(n, grid_splits, inv_splits, least);
  const int valid = n > 0 ? min(grid_splits, (n + chunk - 1) / chunk) : 0;
  float mx = kEmpty;
#pragma unroll
  for (int i = 0; i < kBatch; ++i) mx = fmaxf(mx, i < valid ? ms[i] : kEmpty);
  for (int s = kBatch; s < valid; ++s) mx = fmaxf(mx, part.m[base + s]);
  float lsum = 0.f, o = 0.f;
  for (int s0 = 0; s0 < valid; s0 += kBatch) {
    if (s0) load(s0);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      // a split past the row's end was never written: selected away, not scaled
      const bool live = s0 + i < valid;
      const float f = live ? __builtin_amdgcn_exp2f(ms[i] - mx) : 0.f;
      lsum += live ? ls[i] * f : 0.f;
      o += live ? os[i] * f : 0.f;
    }
  }
  const int64_t at = out_mb ? frag_offset_rows(b, (int64_t)hq * kD + c, out_mb) : (b * q_heads + hq) * kD + c;
  out[at] = (bf16)f32_to_bf16(lsum == 0.f ? 0.f : o / lsum * kBack);
}

int64_t workspace_bytes(int64_t batch, int64_t q_heads, int64_t splits) {
  if (splits <= 1) return 0;
  const int64_t n = batch * q_heads * splits;
  return n * kD * 4 + 2 * align_up(n * 4, 256);
}

template <int kBits, int P, bool kFused, int kWaves>
int launch_sized(const bf16 *q, int64_t qs0, int64_t qs1, const Cache &cache, const int32_t *used, int64_t batch,
                 int64_t q_heads, int64_t kv_heads, int64_t capacity, float scale, int64_t max_len, uint32_t inv_splits,
                 int least, int grid_splits, int stride_splits, const Partial &part, const QkvIn &in, bf16 *out,
                 int out_mb, hipStream_t s) {
  // KV heads fastest: workgroups go to the XCDs in turn, and with the splits fastest one XCD
  // would have the first split of every row and another the last (8 rows of 8191 to 32768
  // positions in four splits 21.5 us against 20.7, three rows of 8 bits in eight 7.65 and 7.5).
  const dim3 grid((unsigned)kv_heads, (unsigned)grid_splits, (unsigned)batch);
  decode_quant_kernel<kBits, P, kFused, kWaves><<<grid, kWaves * kWave, 0, s>>>(
      q, qs0, qs1, cache, used, (int)q_heads, (int)kv_heads, capacity, scale, (int)max_len, inv_splits, least,
      stride_splits, part, in, out, out_mb);
  LM_CHECK_LAUNCH();
  return LM_OK;
}

struct Call {
  int64_t batch, q_heads, kv_heads, capacity, head_dim, max_len, num_splits, bits;
};

// Argument checks of both entry points; *run false where nothing is to launch.
int check_call(const Call &c, bool *run) {
  *run = false;
  LM_REQUIRE(c.batch >= 0 && c.q_heads > 0 && c.kv_heads > 0 && c.q_heads % c.kv_heads == 0 && c.capacity > 0 &&
             c.max_len > 0 && c.num_splits > 0 && c.num_splits <= 1024 && c.max_len < ((int64_t)1 << 30) &&
             c.batch <= 65535 && c.kv_heads <= 65535);
  if (c.head_dim != kD || (c.bits != 4 && c.bits != 8) || c.q_heads / c.kv_heads > 16) return LM_EUNSUPPORTED;
  *run = c.batch > 0;
  return LM_OK;
}

// The fewest positions of a split, `chunk` being one's share of the longest row. A CU holds
// four workgroups in 4 bits and two in 8 (their LDS). While the grid's workgroups all run at
// once, a row far below the plan's bound is cut to single stages, which is the shortest way
// through it: rows of 300 to 1000 positions in eight splits of a plan to 16384, 16 rows x 8
// heads in 4 bits 7.3 us, with 256 positions or more 8.4, 8 rows in 8 bits 7.2 and 7.6 (one
// row of 1000 in sixteen splits 6.2, 6.5, with 512 or more 7.1). Beyond that the pieces
// queue, and a workgroup's four waves get a stage each: 18 rows in 4 bits 8.7 and 8.4, 24
// rows 10.2 and 9.1, fused 12.6 and 11.2; in 8 bits 10 rows 9.1 and 7.7, 20 rows 11.8 and
// 10.5. Rows of 100 to 300 lose there (20 rows in 4 bits 7.0 and 7.9, fused 9.8 and 9.9);
// rows whose pieces are longer anyway do not notice.
int least_chunk(int64_t bits, int64_t workgroups, int chunk) {
  const bool at_once = workgroups <= kCUs * (bits == 4 ? 4 : 2);
  const int wanted = at_once ? kStageKeys : 4 * kStageKeys;
  return chunk < wanted ? chunk : wanted;
}

bool aligned16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

int launch_decode_quant(const Call &c, const void *q, int64_t qs0, int64_t qs1, const Cache &cache,
                        const int32_t *used, float scale, const QkvIn &in, void *out, int out_mb, void *workspace,
                        int64_t workspace_bytes_, void *stream) {
  LM_REQUIRE(aligned16(cache.k) && aligned16(cache.v) && reinterpret_cast<uintptr_t>(cache.scales) % 4 == 0);
  const int64_t need = workspace_bytes(c.batch, c.q_heads, c.num_splits);
  if (need > 0 && (!workspace || workspace_bytes_ < need)) return LM_EWORKSPACE;
  LM_REQUIRE(need == 0 || aligned16(workspace));
  const int chunk = (int)align_up(cdiv(c.max_len, c.num_splits), kStageKeys);
  const int splits = (int)cdiv(c.max_len, chunk);
  const int least = least_chunk(c.bits, (int64_t)splits * c.kv_heads * c.batch, chunk);
  // Rounded up; of no use with one split.
  const uint32_t inv_splits = (uint32_t)((((uint64_t)1 << 32) + splits - 1) / splits);
  Partial part{nullptr, nullptr, nullptr};
  if (splits > 1) {
    const int64_t n = c.batch * c.q_heads * c.num_splits;
    char *w = static_cast<char *>(workspace);
    part.o = reinterpret_cast<float *>(w);
    part.m = reinterpret_cast<float *>(w + n * kD * 4);
    part.l = reinterpret_cast<float *>(w + n * kD * 4 + align_up(n * 4, 256));
  }
  // Partials are indexed with the caller's split count as the stride.
  const int stride_splits = splits > 1 ? (int)c.num_splits : 1;
  hipStream_t s = (hipStream_t)stream;
  const int64_t G = c.q_heads / c.kv_heads;
  auto pick = [&](auto fused, auto bits, auto waves) {
    constexpr bool kFused = decltype(fused)::value;
    constexpr int kBits = decltype(bits)::value, kWaves = decltype(waves)::value;
    auto go = G <= 4   ? launch_sized<kBits, 4, kFused, kWaves>
              : G <= 8 ? launch_sized<kBits, 8, kFused, kWaves>
                       : launch_sized<kBits, 16, kFused, kWaves>;
    return go((const bf16 *)q, qs0, qs1, cache, used, c.batch, c.q_heads, c.kv_heads, c.capacity, scale, c.max_len,
              inv_splits, least, splits, stride_splits, part, in, (bf16 *)out, out_mb, s);
  };
  // Up to one workgroup per CU a wave has its SIMD to itself, and a 4-bit stage's chain
  // of dependent steps (0.57 us) takes longer than its bytes: eight waves where a split of
  // the longest row gives them two stages each. 24 rows to 2000 positions 8.4 us with four,
  // 7.6 with eight; 32 rows to 4095 14.7 and 13.6, 8 rows to 32768 in four splits 26.9 and
  // 21.7; 10 rows to 1000 5.4 and 5.5, one row of 509 3.6 and 3.8. The host knows the bound
  // and not the rows: under a bound of 2000 to 4095 rows of 500 to 1000 take 5.9 to 6.3 us
  // either way, rows of 300 to 500 4.6 to 4.8 with four and 5.0 to 5.3 with eight. In 8 bits
  // they differ by 2 to 4% (32 rows to 4095 22.5 and 21.9), which a second set of kernels is
  // not worth.
  const bool wide = c.bits == 4 && (int64_t)splits * c.kv_heads * c.batch <= kCUs && chunk >= 16 * kStageKeys;
  typedef std::integral_constant<int, 4> Four;
  typedef std::integral_constant<int, 8> Eight;
  auto run = [&](auto fused) {
    return c.bits == 8 ? pick(fused, Eight{}, Four{})
           : wide      ? pick(fused, Four{}, Eight{})
                       : pick(fused, Four{}, Four{});
  };
  const int status = in.part ? run(std::true_type{}) : run(std::false_type{});
  if (status != LM_OK || splits == 1) return status;
  auto combine = splits <= 4   ? decode_quant_combine_kernel<4>
                 : splits <= 8 ? decode_quant_combine_kernel<8>
                               : decode_quant_combine_kernel<16>;
  combine<<<dim3((unsigned)cdiv(c.q_heads, kCombineHeads), (unsigned)c.batch), kCombineHeads * kD, 0, s>>>(
      used, (int)c.q_heads, c.capacity, (int)c.max_len, inv_splits, least, splits, stride_splits, part,
      (bf16 *)out, out_mb);
  LM_CHECK_LAUNCH();
  return LM_OK;
}

}  // namespace
}  // namespace lm

using namespace lm;

extern "C" int lm_flash_decode_quant(const void *q, int64_t qs0, int64_t qs1, const void *k_codes,
                                     const void *v_codes, const void *scales, const int32_t *used,
                                     int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t capacity,
                                     int64_t head_dim, int64_t bits, float scale, int64_t max_len,
                                     int64_t num_splits, void *out, void *workspace,
                                     int64_t workspace_bytes_, void *stream) {
  const Call c{batch, q_heads, kv_heads, capacity, head_dim, max_len, num_splits, bits};
  bool run;
  const int status = check_call(c, &run);
  if (status != LM_OK || !run) return status;
  LM_REQUIRE(q && k_codes && v_codes && scales && used && out);
  LM_REQUIRE(aligned16(q) && qs0 % 8 == 0 && qs1 % 8 == 0);
  const Cache cache{(uint8_t *)const_cast<void *>(k_codes), (uint8_t *)const_cast<void *>(v_codes),
                    (uint32_t *)const_cast<void *>(scales)};
  const QkvIn in{nullptr, 0, nullptr, 0, nullptr, nullptr, nullptr};
  return launch_decode_quant(c, q, qs0, qs1, cache, used, scale, in, out, 0, workspace, workspace_bytes_, stream);
}

extern "C" int lm_flash_decode_quant_qkv(const float *qkv_partials, int64_t qkv_splits, const void *cos_sin,
                                         int64_t table_len, const int64_t *positions,
                                         const uint8_t *active, void *k_codes, void *v_codes, void *scales,
                                         const int32_t *used, const int32_t *row_order, int64_t batch,
                                         int64_t q_heads, int64_t kv_heads, int64_t capacity,
                                         int64_t head_dim, int64_t bits, float scale, int64_t max_len,
                                         int64_t num_splits, int frag_out, void *out, void *workspace,
                                         int64_t workspace_bytes_, void *stream) {
  const Call c{batch, q_heads, kv_heads, capacity, head_dim, max_len, num_splits, bits};
  bool run;
  const int status = check_call(c, &run);
  if (status != LM_OK) return status;
  LM_REQUIRE(qkv_splits >= 1 && table_len > 0);
  if (qkv_splits > kMaxQkvSplits || (frag_out && batch > 128)) return LM_EUNSUPPORTED;
  if (!run) return LM_OK;
  LM_REQUIRE(qkv_partials && cos_sin && positions && k_codes && v_codes && scales && used && out);
  LM_REQUIRE(aligned16(qkv_partials));
  const QkvIn in{qkv_partials, (int)qkv_splits, (const bf16 *)cos_sin, table_len, positions, active, row_order};
  const Cache cache{(uint8_t *)k_codes, (uint8_t *)v_codes, (uint32_t *)scales};
  return launch_decode_quant(c, nullptr, 0, 0, cache, used, scale, in, out, frag_out ? frag_row_blocks(batch) : 0,
                             workspace, workspace_bytes_, stream);
}
