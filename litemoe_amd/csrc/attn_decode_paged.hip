// Split-K decode attention over the paged KV cache on the matrix cores:
//   out[b, h] = softmax_j(scale q_h . K_j) V,  j < used[b].
//
// Workgroup (kv head, split, row); its waves take the split's tiles of 32
// positions in turn, each wave its own, without barriers, with two tiles of K and
// V in registers on their way. A tile is two halves of 16 positions, and a page
// holds a multiple of 16, so a half lies in one page: its number is a scalar load
// two tiles ahead, and the lanes' offsets from the half's first position are
// constants. Every KV byte is read once, straight into MFMA operands.
//
// Scores: S = K . q^T with v_mfma_f32_16x16x32_bf16, A the 16 positions of a half
// (lane l: position l % 16, 16 bytes of channels), B the query heads of the KV head
// (column l % 16; columns past the G heads are zero). Lane l then holds positions
// 4 (l / 16) .. + 3 of both halves for query head l % 16.
//
// P.V: O^T = V^T . P^T. The sum over positions may take them in any order that both
// operands share, so a lane's eight probabilities are its B operand as they stand: k
// index 8 g + i is position 4 g + i of half 0, and 8 g + 4 + i that of half 1. A is
// V transposed: lane l loads channels D/16 (l % 16) .. of those eight positions
// (8 or 16 bytes each, rows of one position contiguous over 16 lanes) and pairs
// them per channel with v_perm, 2 instructions a position and 64 bytes. A row of
// the result is then a channel of the same 16-fold stride, and the lane's
// accumulators are D/4 consecutive channels. The row sums of P come from one more
// MFMA with ones, so they sum the probabilities as they were rounded.
//
// The running maximum is a column's own reference, kept kAbove over the score that
// set it and moved only when a score passes it, so nothing crosses lanes in the
// usual tile. Waves merge through LDS, splits by log-sum-exp in a second launch.
//
// Masked positions (past used[b], or in no page) may hold anything: their scores
// become -inf and their V words 0. Only a row's last tile and tiles with a page
// missing take that path.
//
// Reference semantics: litemoe/flash_decode.py:16-22; masking litemoe/cache.py:42-47.
#include "paged.h"

#include <type_traits>

namespace lm {
namespace {

constexpr int kTile = 32;
constexpr int kWaves = 4;
constexpr int kThreads = kWaves * kWave;
constexpr int kMaxQkvSplits = 8;
constexpr int kMaxGroups = 16;

// Running maximum before any position: below every finite score, and finite, so
// exp2(kEmpty - m) and exp2(-inf - kEmpty) are 0.
constexpr float kEmpty = -3.402823466e38f;
constexpr float kAbove = 8.f;

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

struct Partial {
  float *o;   // [batch, q_heads, splits, D]
  float *m;   // [batch, q_heads, splits]
  float *l;   // sums of the rounded probabilities, as m
  float *lw;  // weighed: sums of the probabilities, as m
  float *s;   // weighed: scores in log2 units, [batch, q_heads, padded]
  int64_t padded;
};

struct QkvIn {
  const float *part;  // [splits][batch][(q_heads + 2 kv_heads) D], NULL: unfused
  int splits;
  Rotation rot;
  const int64_t *pos;
  const uint8_t *active;
  const int32_t *order;
};

struct Shape {
  int q_heads, G, max_len, splits;
  float scale;
  int64_t batch;
};

// Positions of row b that are looked at.
__device__ __forceinline__ int row_length(int used, const Shape &sh, const PagedKV &kv) {
  return max(0, min(min(used, sh.max_len), kv.width << kv.shift));
}
// Splits that hold a tile of a row of n positions: tiles go to the waves of all
// splits in turn, kWaves a split.
__device__ __forceinline__ int row_splits(int n, const Shape &sh) {
  return min(sh.splits, (n + kTile * kWaves - 1) / (kTile * kWaves));
}

template <int D>
struct Kv {
  typedef typename std::conditional<D == 64, u32x2, u32x4>::type V;
  u32x4 k[2][D / 32];
  V v[2][4];
  bool ok[2];  // the half's page exists
};

__device__ __forceinline__ int scalar(int v) { return __builtin_amdgcn_readfirstlane(v); }

// A uniform word of memory that this launch does not write, through the constant
// cache: it does not count with the vector loads in flight.
template <typename T>
__device__ __forceinline__ T constant(const T *p) {
  return *(const __attribute__((address_space(4))) T *)p;
}

template <int D, bool kFused, bool kWeigh>
__global__ void __launch_bounds__(kWaves *kWave, D == 64 ? 4 : 2)
decode_paged_kernel(const bf16 *__restrict__ q, int64_t qs0, int64_t qs1, PagedKV kv,
                    const int32_t *__restrict__ table, const int32_t *__restrict__ used, Shape sh, Partial part,
                    QkvIn in, bf16 *__restrict__ out, int out_mb) {
  constexpr int kSteps = D / 32, kCh = D / 16;  // k steps of a score; channels a lane takes of a V row
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int h = blockIdx.x, split = blockIdx.y;
  const int64_t b = kFused && in.order ? constant(in.order + blockIdx.z) : blockIdx.z;
  const int lane = threadIdx.x % kWave, wave = scalar(threadIdx.x / kWave);
  const int r = lane & 15, g = lane >> 4;
  const int G = sh.G;

  // Fused: loads of the partials first, so that nothing of the KV stream stands before them.
  const int ncols = (sh.q_heads + 2 * kv.heads) * D;
  const int stages = (G + 2) * (D / 4);  // threads' work staging 4 channels each
  f32x4 pv[kMaxQkvSplits];
  auto source = [&](int t) {
    const int hs = t / (D / 4), c4 = t % (D / 4) * 4;
    const int head = hs < G ? h * G + hs : (hs == G ? sh.q_heads + h : sh.q_heads + kv.heads + h);
    return in.part + b * ncols + (int64_t)head * D + c4;
  };
  // and the angles of pair threadIdx.x % (D / 2), the pair that the thread turns.
  constexpr int kPairs = D / 2;
  static_assert(kThreads % kPairs == 0, "a thread turns one pair of every head it takes");
  const int pair = threadIdx.x % kPairs, half = in.rot.rotary / 2;
  bool in_table = false, writes = false;
  float turn_c = 1.f, turn_s = 0.f;
  u32x4 qw[kSteps];
  if constexpr (kFused) {
    if ((int)threadIdx.x < stages) {
      const float *src = source(threadIdx.x);
#pragma unroll
      for (int s = 0; s < kMaxQkvSplits; ++s)
        if (s < in.splits) pv[s] = *reinterpret_cast<const f32x4 *>(src + (int64_t)s * sh.batch * ncols);
    }
    const int64_t p = constant(in.pos + b);
    in_table = p >= 0 && p < in.rot.table_len;
    const int64_t at = (in_table ? p : 0) * in.rot.rotary + (pair < half ? pair : 0);
    if (in.rot.f32) {
      turn_c = static_cast<const float *>(in.rot.table)[at];
      turn_s = static_cast<const float *>(in.rot.table)[at + half];
    } else {
      turn_c = bf16_to_f32(static_cast<const bf16 *>(in.rot.table)[at]);
      turn_s = bf16_to_f32(static_cast<const bf16 *>(in.rot.table)[at + half]);
    }
    writes = !in.active || in.active[b];
  } else {
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
      qw[s] = r < G ? *reinterpret_cast<const u32x4 *>(q + b * qs0 + (int64_t)(h * G + r) * qs1 + 32 * s + 8 * g)
                    : u32x4{0, 0, 0, 0};
  }

  const int first = split * kWaves + wave, stride = sh.splits * kWaves;  // this wave's tiles
  const int32_t *row_table = table + b * kv.width;
  const uint32_t k_off = (uint32_t)(r * D + g * 8) * 2, v_off = (uint32_t)(4 * g * D + r * kCh) * 2;
  const int page_mask = (1 << kv.shift) - 1;
  struct Ids {
    int id[2];
  };
  auto ids_of = [&](int tile) {
    Ids x;
    const int j = tile * kTile;
#pragma unroll
    for (int t = 0; t < 2; ++t) x.id[t] = constant(row_table + min((j + 16 * t) >> kv.shift, kv.width - 1));
    return x;
  };
  const Ids ia = ids_of(first), ib = ids_of(first + stride);
  const int held = constant(used + b), n = row_length(held, sh, kv);
  const int tiles = (n + kTile - 1) / kTile;
  if (split * kWaves >= tiles) {
    // nothing of this row here: with one split its zeros are written
    if (sh.splits == 1) {
      for (int t = threadIdx.x; t < G * D; t += kThreads) {
        const int hq = h * G + t / D, c = t % D;
        out[out_mb ? frag_offset_rows(b, (int64_t)hq * D + c, out_mb) : (b * sh.q_heads + hq) * D + c] = 0;
      }
    }
    return;
  }

  // In bounds whatever the table holds: a page that does not exist, and a tile past the
  // row's end, are read from page 0. So the table's words need not wait for the length.
  auto load = [&](Kv<D> &x, const Ids &ids, int tile) {
    const int j = tile * kTile;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int id = ids.id[t];
      x.ok[t] = (uint32_t)id < (uint32_t)kv.pages;
      const int64_t from =
          ((((int64_t)(x.ok[t] && tile < tiles ? id : 0) * kv.heads + h) << kv.shift) + ((j + 16 * t) & page_mask)) * D;
      const char *kb = reinterpret_cast<const char *>(kv.k + from), *vb = reinterpret_cast<const char *>(kv.v + from);
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
        x.k[t][s] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(kb + k_off + 64 * s));
#pragma unroll
      for (int i = 0; i < 4; ++i)
        x.v[t][i] = __builtin_nontemporal_load(reinterpret_cast<const typename Kv<D>::V *>(vb + v_off + 2 * D * i));
    }
  };
  // The first two tiles are on their way before anything else is waited for, without a
  // branch: loads under one would make the wait counts fall back to waiting for all.
  Kv<D> xa, xb;
  load(xa, ia, first);
  load(xb, ib, first + stride);
  Ids na = ids_of(first + 2 * stride), nb = ids_of(first + 3 * stride);

  // The query heads as B operands; fused, also the new key and value (rows G and
  // G + 1 of sm_rot), rotated and rounded.
  uint16_t(*sm_rot)[D] = reinterpret_cast<uint16_t(*)[D]>(smem);
  bool own = false;  // this split holds the new token, which is stored and attended from sm_rot
  int64_t new_cell = 0;
  if constexpr (kFused) {
    float(*sm_x)[D] = reinterpret_cast<float(*)[D]>(smem + (G + 2) * D * 2);
    auto stage = [&](int t, f32x4 sum) {
      const int hs = t / (D / 4), c4 = t % (D / 4) * 4;
#pragma unroll
      for (int i = 0; i < 4; ++i) sm_x[hs][c4 + i] = in.rot.f32 ? sum[i] : round_bf16(sum[i]);
    };
    if ((int)threadIdx.x < stages) {
      f32x4 sum = pv[0];
#pragma unroll
      for (int s = 1; s < kMaxQkvSplits; ++s)
        if (s < in.splits) sum += pv[s];
      stage(threadIdx.x, sum);
    }
    for (int t = threadIdx.x + kThreads; t < stages; t += kThreads) {
      const float *src = source(t);
      f32x4 sum = *reinterpret_cast<const f32x4 *>(src);
      for (int s = 1; s < in.splits; ++s)
        sum += *reinterpret_cast<const f32x4 *>(src + (int64_t)s * sh.batch * ncols);
      stage(t, sum);
    }
    __syncthreads();
    // Pair i of a head: the rotation's pairs first, then the channels past them in twos.
    const bool spread = pair < half && in.rot.neox;
    const int c1 = spread ? pair : 2 * pair, c2 = spread ? pair + half : 2 * pair + 1;
    for (int hs = threadIdx.x / kPairs; hs < G + 2; hs += kThreads / kPairs) {
      const float x1 = sm_x[hs][c1], x2 = sm_x[hs][c2];
      float o1 = x1, o2 = x2;
      if (in_table && hs <= G && pair < half) turn_pair(in.rot.f32, x1, x2, turn_c, turn_s, o1, o2);
      sm_rot[hs][c1] = (uint16_t)f32_to_bf16(o1);
      sm_rot[hs][c2] = (uint16_t)f32_to_bf16(o2);
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
      qw[s] = r < G ? *reinterpret_cast<const u32x4 *>(&sm_rot[r][32 * s + 8 * g]) : u32x4{0, 0, 0, 0};
    // The new token's place is the row's last, if the row was not cut short.
    const int last = n - 1;
    if (writes && held == n && (tiles - 1) / kWaves % sh.splits == split) {
      const int id = constant(row_table + (last >> kv.shift));
      own = (uint32_t)id < (uint32_t)kv.pages;
      new_cell = ((((int64_t)(own ? id : 0) * kv.heads + h) << kv.shift) + (last & page_mask)) * D;
    }
  }

  const float sl2 = sh.scale * 1.4426950408889634f;
  float m = kEmpty, lw = 0.f;
  f32x4 l{0.f, 0.f, 0.f, 0.f}, acc[kCh];
#pragma unroll
  for (int c = 0; c < kCh; ++c) acc[c] = f32x4{0.f, 0.f, 0.f, 0.f};
  const u32x4 ones{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};

  auto compute = [&](Kv<D> &x, int tile) {
    const int left = n - tile * kTile;  // positions of the row from this tile on
    const bool edge = left < kTile || (kFused && own && tile == tiles - 1) || !x.ok[0] || !x.ok[1];
    if (kFused && own && tile == tiles - 1) {
      // The new key and value take the place of what was loaded.
      const int at = left - 1;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if (t * 16 + r == at) {
#pragma unroll
          for (int s = 0; s < kSteps; ++s) x.k[t][s] = *reinterpret_cast<const u32x4 *>(&sm_rot[G][32 * s + 8 * g]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (t * 16 + 4 * g + i == at)
            x.v[t][i] = *reinterpret_cast<const typename Kv<D>::V *>(&sm_rot[G + 1][r * kCh]);
      }
    }
    f32x4 c[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      c[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < kSteps; ++s) c[t] = mfma16x16x32(x.k[t][s], qw[s], c[t]);
    }
    float sc[2][4];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) sc[t][i] = c[t][i] * sl2;
    if (edge) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool ok = x.ok[t] && t * 16 + 4 * g + i < left;
          sc[t][i] = ok ? sc[t][i] : -INFINITY;
#pragma unroll
          for (int w = 0; w < kCh / 2; ++w) x.v[t][i][w] = ok ? x.v[t][i][w] : 0u;
        }
    }
    if constexpr (kWeigh) {
      if (r < G) {
        float *to = part.s + (b * sh.q_heads + h * G + r) * part.padded + (int64_t)tile * kTile + 4 * g;
#pragma unroll
        for (int t = 0; t < 2; ++t)
          *reinterpret_cast<f32x4 *>(to + 16 * t) = f32x4{sc[t][0], sc[t][1], sc[t][2], sc[t][3]};
      }
    }
    float mx = sc[0][0];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) mx = fmaxf(mx, sc[t][i]);
    if (__any(mx > m)) {
      mx = fmaxf(mx, xor_lanes<16>(mx));
      mx = fmaxf(mx, xor_lanes<32>(mx));
      const bool up = mx > m;
      const float to = mx + kAbove;
      const float f = up ? __builtin_amdgcn_exp2f(m - to) : 1.f;
      m = up ? to : m;
      lw *= f;
      l *= f;
#pragma unroll
      for (int cb = 0; cb < kCh; ++cb) acc[cb] *= f;
    }
    u32x4 p;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float p0 = __builtin_amdgcn_exp2f(sc[t][2 * i] - m), p1 = __builtin_amdgcn_exp2f(sc[t][2 * i + 1] - m);
        if constexpr (kWeigh) {
          lw += p0;
          lw += p1;
        }
        p[2 * t + i] = pack_bf16_nc(p0, p1);
      }
    l = mfma16x16x32(ones, p, l);
#pragma unroll
    for (int cb = 0; cb < kCh; ++cb) {
      const uint32_t sel = cb % 2 ? 0x07060302u : 0x05040100u;
      u32x4 vt;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          vt[2 * t + i] = __builtin_amdgcn_perm(x.v[t][2 * i + 1][cb / 2], x.v[t][2 * i][cb / 2], sel);
      acc[cb] = mfma16x16x32(vt, p, acc[cb]);
    }
  };

  // Tiles in pairs while there is one to load for the first of the two; the second may
  // be past the row's end, once.
  int tile = first;
  for (; tile + 2 * stride < tiles; tile += 2 * stride) {
    compute(xa, tile);
    load(xa, na, tile + 2 * stride);
    compute(xb, tile + stride);
    load(xb, nb, tile + 3 * stride);
    na = ids_of(tile + 4 * stride);
    nb = ids_of(tile + 5 * stride);
  }
  if (tile < tiles) compute(xa, tile);
  if (tile + stride < tiles) compute(xb, tile + stride);

  if constexpr (kFused) {
    // Stored behind the stream, which does not wait for it.
    if (own && (int)threadIdx.x < D / 4) {
      const int side = threadIdx.x / (D / 8), c = threadIdx.x % (D / 8) * 8;
      *reinterpret_cast<u32x4 *>((side ? kv.v : kv.k) + new_cell + c) =
          *reinterpret_cast<const u32x4 *>(&sm_rot[G + side][c]);
    }
    __syncthreads();  // sm_rot is done with
  }
  if constexpr (kWeigh) {
    lw += xor_lanes<16>(lw);
    lw += xor_lanes<32>(lw);
  }
  // Waves merge: [wave][G][D] accumulators, then [wave][G] of m, l and lw.
  float *sm_o = reinterpret_cast<float *>(smem);
  float *sm_m = sm_o + kWaves * G * D, *sm_l = sm_m + kWaves * G, *sm_w = sm_l + kWaves * G;
  if (r < G) {
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
      for (int cb = 0; cb < kCh; cb += 4)
        *reinterpret_cast<f32x4 *>(sm_o + (wave * G + r) * D + (4 * g + x) * kCh + cb) =
            f32x4{acc[cb][x], acc[cb + 1][x], acc[cb + 2][x], acc[cb + 3][x]};
    if (g == 0) {
      sm_m[wave * G + r] = m;
      sm_l[wave * G + r] = l[0];
      if constexpr (kWeigh) sm_w[wave * G + r] = lw;
    }
  }
  __syncthreads();
  for (int t = threadIdx.x; t < G * D; t += kThreads) {
    const int gh = t / D, c = t % D;
    float mx = sm_m[gh];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) mx = fmaxf(mx, sm_m[w * G + gh]);
    float lsum = 0.f, wsum = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float f = __builtin_amdgcn_exp2f(sm_m[w * G + gh] - mx);
      lsum += sm_l[w * G + gh] * f;
      if constexpr (kWeigh) wsum += sm_w[w * G + gh] * f;
      o += sm_o[(w * G + gh) * D + c] * f;
    }
    const int hq = h * G + gh;
    const int64_t at = (b * sh.q_heads + hq) * sh.splits + split;
    if (sh.splits == 1) {
      out[out_mb ? frag_offset_rows(b, (int64_t)hq * D + c, out_mb) : (b * sh.q_heads + hq) * D + c] =
          (bf16)f32_to_bf16(lsum == 0.f ? 0.f : o / lsum);
    } else {
      part.o[at * D + c] = o;
    }
    if (c == 0 && (kWeigh || sh.splits > 1)) {
      part.m[at] = mx;
      part.l[at] = lsum;
      if constexpr (kWeigh) part.lw[at] = wsum;
    }
  }
}

// grid (groups of query heads, batch), one thread per channel: the splits'
// partials by log-sum-exp, those of kBatch splits requested together.
constexpr int kCombineHeads = 2;
template <int D, int kBatch>
__global__ void __launch_bounds__(kCombineHeads *D)
decode_paged_combine_kernel(const int32_t *__restrict__ used, Shape sh, PagedKV kv, Partial part,
                            bf16 *__restrict__ out, int out_mb) {
  const int hq = blockIdx.x * kCombineHeads + threadIdx.x / D;
  if (hq >= sh.q_heads) return;
  const int64_t b = blockIdx.y;
  const int c = threadIdx.x % D;
  const int64_t base = (b * sh.q_heads + hq) * sh.splits;
  float ms[kBatch], ls[kBatch], os[kBatch];
  auto load = [&](int s0) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int64_t at = base + min(s0 + i, sh.splits - 1);
      ms[i] = part.m[at];
      ls[i] = part.l[at];
      os[i] = part.o[at * D + c];
    }
  };
  load(0);
  const int valid = row_splits(row_length(used[b], sh, kv), sh);
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
  const int64_t at = out_mb ? frag_offset_rows(b, (int64_t)hq * D + c, out_mb) : (b * sh.q_heads + hq) * D + c;
  out[at] = (bf16)f32_to_bf16(lsum == 0.f ? 0.f : o / lsum);
}

// after[b, h, j] = before[b, h, j] + sum over the KV head's query heads of their
// probability of position j, j < the row's length. A thread four positions. With
// splits the first workgroup of a (row, KV head) also joins their results, in place of
// the launch above.
constexpr int kWeighThreads = 256, kWeighSpan = 4 * kWeighThreads, kAhead = 4;
template <int D>
__global__ void __launch_bounds__(kWeighThreads)
weigh_kernel(const int32_t *__restrict__ used, Shape sh, PagedKV kv, Partial part, const float *before, float *after,
             bf16 *__restrict__ out, int out_mb) {
  __shared__ float sm_m[kMaxGroups], sm_f[kMaxGroups];
  const int h = blockIdx.y, G = sh.G;
  const int64_t b = blockIdx.z;
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int n = row_length(used[b], sh, kv), valid = row_splits(n, sh);
  const int j = (blockIdx.x * kWeighThreads + threadIdx.x) * 4;
  const bool joins = blockIdx.x == 0 && sh.splits > 1;
  if ((int)blockIdx.x * kWeighSpan >= n && !joins) return;
  // The scores and weights of this thread's positions are on their way while the
  // heads' sums are joined. The buffers hold a multiple of 16 positions a row.
  const float *sc = part.s + (b * sh.q_heads + h * G) * part.padded + j;
  const int64_t at = (b * kv.heads + h) * ((int64_t)kv.width << kv.shift) + j;
  f32x4 s[kAhead], old{0.f, 0.f, 0.f, 0.f};
  if (j < n) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) s[i] = *reinterpret_cast<const f32x4 *>(sc + min(i, G - 1) * part.padded);
    old = *reinterpret_cast<const f32x4 *>(before + at);
  }
  for (int gh = wave; gh < G; gh += kWeighThreads / kWave) {
    const int64_t base = (b * sh.q_heads + h * G + gh) * sh.splits;
    float mx = kEmpty, l = 0.f;
    for (int s0 = lane; s0 < valid; s0 += kWave) mx = fmaxf(mx, part.m[base + s0]);
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) mx = fmaxf(mx, shfl_xor(mx, d));
    for (int s0 = lane; s0 < valid; s0 += kWave) l += part.lw[base + s0] * __builtin_amdgcn_exp2f(part.m[base + s0] - mx);
    l = wave_sum(l);
    if (lane == 0) {
      sm_m[gh] = mx;
      sm_f[gh] = l == 0.f ? 0.f : 1.f / l;
    }
  }
  __syncthreads();
  if (joins) {
    for (int t = threadIdx.x; t < G * D; t += kWeighThreads) {
      const int gh = t / D, c = t % D, hq = h * G + gh;
      const int64_t base = (b * sh.q_heads + hq) * sh.splits;
      float lsum = 0.f, o = 0.f;
#pragma unroll 4
      for (int i = 0; i < valid; ++i) {
        const float f = __builtin_amdgcn_exp2f(part.m[base + i] - sm_m[gh]);
        lsum += part.l[base + i] * f;
        o += part.o[(base + i) * D + c] * f;
      }
      out[out_mb ? frag_offset_rows(b, (int64_t)hq * D + c, out_mb) : (b * sh.q_heads + hq) * D + c] =
          (bf16)f32_to_bf16(lsum == 0.f ? 0.f : o / lsum);
    }
  }
  if (j >= n) return;
  float w[4] = {0.f, 0.f, 0.f, 0.f};
  for (int g0 = 0; g0 < G; g0 += kAhead) {
    if (g0) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) s[i] = *reinterpret_cast<const f32x4 *>(sc + min(g0 + i, G - 1) * part.padded);
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (g0 + i >= G) break;
      const float m = sm_m[g0 + i], f = sm_f[g0 + i];
#pragma unroll
      for (int x = 0; x < 4; ++x) w[x] += __builtin_amdgcn_exp2f(s[i][x] - m) * f;
    }
  }
  if (j + 4 <= n) {
    *reinterpret_cast<f32x4 *>(after + at) = f32x4{old[0] + w[0], old[1] + w[1], old[2] + w[2], old[3] + w[3]};
  } else {
#pragma unroll
    for (int x = 0; x < 4; ++x)
      if (j + x < n) after[at + x] = old[x] + w[x];
  }
}

struct Call {
  int64_t batch, q_heads, kv_heads, head_dim, width, pages, page, max_len, num_splits;
};

int64_t padded_scores(int64_t max_len) { return align_up(max_len, kTile); }

int64_t workspace_bytes(int64_t batch, int64_t q_heads, int64_t head_dim, int64_t max_len, int64_t splits,
                        bool weighed) {
  if (splits <= 1 && !weighed) return 0;
  const int64_t n = batch * q_heads * splits;
  return (splits > 1 ? n * head_dim * 4 : 0) + (weighed ? 3 : 2) * align_up(n * 4, 256) +
         (weighed ? batch * q_heads * padded_scores(max_len) * 4 : 0);
}

// Argument checks of both entry points; *run false where nothing is to launch.
int check_call(const Call &c, bool *run) {
  *run = false;
  LM_REQUIRE(c.batch >= 0 && c.q_heads > 0 && c.kv_heads > 0 && c.q_heads % c.kv_heads == 0 && c.max_len > 0 &&
             c.num_splits > 0 && c.num_splits <= 1024 && c.max_len < ((int64_t)1 << 30) && c.batch <= 65535 &&
             c.kv_heads <= 65535);
  const int status = paged_args_ok(c.width, c.pages, c.page, c.head_dim);
  if (status != LM_OK) return status;
  if (c.q_heads / c.kv_heads > kMaxGroups) return LM_EUNSUPPORTED;
  *run = c.batch > 0;
  return LM_OK;
}

template <int D, bool kFused, bool kWeigh>
int launch_sized(const Call &c, const bf16 *q, int64_t qs0, int64_t qs1, const PagedKV &kv, const int32_t *table,
                 const int32_t *used, const Shape &sh, const Partial &part, const QkvIn &in, bf16 *out, int out_mb,
                 const float *before, float *after, hipStream_t s) {
  // KV heads fastest: workgroups go to the XCDs in turn, so that each XCD has a share
  // of every split.
  const dim3 grid((unsigned)c.kv_heads, (unsigned)sh.splits, (unsigned)c.batch);
  const size_t merge = (size_t)kWaves * sh.G * (D + 3) * 4;
  const size_t rot = kFused ? (size_t)(sh.G + 2) * D * (2 + 4) : 0;
  decode_paged_kernel<D, kFused, kWeigh><<<grid, kWaves * kWave, merge > rot ? merge : rot, s>>>(
      q, qs0, qs1, kv, table, used, sh, part, in, out, out_mb);
  LM_CHECK_LAUNCH();
  if (!kWeigh && sh.splits > 1) {
    auto combine = sh.splits <= 4   ? decode_paged_combine_kernel<D, 4>
                   : sh.splits <= 8 ? decode_paged_combine_kernel<D, 8>
                                    : decode_paged_combine_kernel<D, 16>;
    combine<<<dim3((unsigned)cdiv(c.q_heads, kCombineHeads), (unsigned)c.batch), kCombineHeads * D, 0, s>>>(
        used, sh, kv, part, out, out_mb);
    LM_CHECK_LAUNCH();
  }
  if (kWeigh) {
    weigh_kernel<D><<<dim3((unsigned)cdiv(sh.max_len, kWeighSpan), (unsigned)c.kv_heads, (unsigned)c.batch),
                      kWeighThreads, 0, s>>>(used, sh, kv, part, before, after, out, out_mb);
    LM_CHECK_LAUNCH();
  }
  return LM_OK;
}

int launch_decode_paged(const Call &c, const void *q, int64_t qs0, int64_t qs1, void *k_pages, void *v_pages,
                        const int32_t *table, const int32_t *used, float scale, const QkvIn &in, void *out,
                        int out_mb, const float *before, float *after, void *workspace, int64_t workspace_bytes_,
                        void *stream) {
  LM_REQUIRE(aligned16(k_pages) && aligned16(v_pages) && (before == nullptr) == (after == nullptr) &&
             aligned16(before) && aligned16(after));
  const bool weighed = after != nullptr;
  // No row is longer than the table; what the plan allows beyond it needs no split.
  const int64_t room = c.width * c.page, longest = c.max_len < room ? c.max_len : room;
  const int64_t need = workspace_bytes(c.batch, c.q_heads, c.head_dim, c.max_len, c.num_splits, weighed);
  if (need > 0 && (!workspace || workspace_bytes_ < need)) return LM_EWORKSPACE;
  LM_REQUIRE(need == 0 || aligned16(workspace));
  const int64_t splits = c.num_splits < cdiv(longest, kTile) ? c.num_splits : cdiv(longest, kTile);
  Partial part{nullptr, nullptr, nullptr, nullptr, nullptr, padded_scores(c.max_len)};
  const int64_t n = c.batch * c.q_heads * splits;
  char *w = static_cast<char *>(workspace);
  auto take = [&](int64_t bytes) {
    float *at = reinterpret_cast<float *>(w);
    w += bytes;
    return at;
  };
  if (weighed) part.s = take(c.batch * c.q_heads * part.padded * 4);
  if (splits > 1) part.o = take(n * c.head_dim * 4);
  if (splits > 1 || weighed) {
    part.m = take(align_up(n * 4, 256));
    part.l = take(align_up(n * 4, 256));
    if (weighed) part.lw = take(align_up(n * 4, 256));
  }
  const PagedKV kv{(bf16 *)k_pages, (bf16 *)v_pages, c.pages, (int)c.width, page_shift(c.page), (int)c.kv_heads};
  const int G = (int)(c.q_heads / c.kv_heads);
  const Shape sh{(int)c.q_heads, G, (int)longest, (int)splits, scale, c.batch};
  auto go = [&](auto dim, auto fused, auto weigh) {
    return launch_sized<decltype(dim)::value, decltype(fused)::value, decltype(weigh)::value>(
        c, (const bf16 *)q, qs0, qs1, kv, table, used, sh, part, in, (bf16 *)out, out_mb, before, after,
        (hipStream_t)stream);
  };
  auto sized = [&](auto fused, auto weigh) {
    return c.head_dim == 64 ? go(std::integral_constant<int, 64>{}, fused, weigh)
                            : go(std::integral_constant<int, 128>{}, fused, weigh);
  };
  if (in.part) return weighed ? sized(std::true_type{}, std::true_type{}) : sized(std::true_type{}, std::false_type{});
  return weighed ? sized(std::false_type{}, std::true_type{}) : sized(std::false_type{}, std::false_type{});
}

}  // namespace
}  // namespace lm

using namespace lm;

extern "C" int lm_flash_decode_paged_workspace_size(int64_t batch, int64_t q_heads, int64_t head_dim, int64_t max_len,
                                                    int64_t num_splits, int weighed, int64_t *bytes) {
  LM_REQUIRE(bytes && batch >= 0 && q_heads > 0 && max_len > 0 && num_splits > 0);
  if (head_dim != 64 && head_dim != 128) return LM_EUNSUPPORTED;
  *bytes = workspace_bytes(batch, q_heads, head_dim, max_len, num_splits, weighed != 0);
  return LM_OK;
}

extern "C" int lm_flash_decode_paged(const lm_flash_decode_paged_args *args, void *stream) {
  LM_REQUIRE(args);
  const auto &a = *args;
  const Call c{a.batch, a.q_heads, a.kv_heads, a.head_dim, a.width, a.pages, a.page, a.max_len, a.num_splits};
  bool run;
  const int status = check_call(c, &run);
  if (status != LM_OK || !run) return status;
  LM_REQUIRE(a.q && a.k_pages && a.v_pages && a.block_table && a.used && a.out);
  LM_REQUIRE(aligned16(a.q) && a.qs0 % 8 == 0 && a.qs1 % 8 == 0);
  const QkvIn in{nullptr, 0, {nullptr, 0, 0, false, false}, nullptr, nullptr, nullptr};
  return launch_decode_paged(c, a.q, a.qs0, a.qs1, const_cast<void *>(a.k_pages), const_cast<void *>(a.v_pages),
                             a.block_table, a.used, (float)a.scale, in, a.out, 0, a.weights, a.weights_out, a.workspace,
                             a.workspace_bytes, stream);
}

extern "C" int lm_flash_decode_paged_qkv(const lm_flash_decode_paged_qkv_args *args, void *stream) {
  LM_REQUIRE(args);
  const auto &a = *args;
  const Call c{a.batch, a.q_heads, a.kv_heads, a.head_dim, a.width, a.pages, a.page, a.max_len, a.num_splits};
  bool run;
  const int status = check_call(c, &run);
  if (status != LM_OK) return status;
  LM_REQUIRE(a.qkv_splits >= 1);
  if (a.qkv_splits > kMaxQkvSplits || (a.frag_out && a.batch > 128)) return LM_EUNSUPPORTED;
  if (!run) return LM_OK;
  LM_REQUIRE(a.qkv_partials && a.positions && a.k_pages && a.v_pages && a.block_table && a.used && a.out);
  LM_REQUIRE(aligned16(a.qkv_partials) && rotation_ok(a.cos_sin, a.table_len, a.rotary, a.head_dim));
  const Rotation rot{a.cos_sin, a.table_len, (int)a.rotary, a.table_f32 != 0, a.neox != 0};
  const QkvIn in{a.qkv_partials, (int)a.qkv_splits, rot, a.positions, a.active, a.row_order};
  return launch_decode_paged(c, nullptr, 0, 0, a.k_pages, a.v_pages, a.block_table, a.used, (float)a.scale, in, a.out,
                             a.frag_out ? frag_row_blocks(a.batch) : 0, a.weights, a.weights_out, a.workspace,
                             a.workspace_bytes, stream);
}
