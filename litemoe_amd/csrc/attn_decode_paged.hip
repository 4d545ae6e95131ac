// Decode attention over the paged KV cache on the matrix cores:
//   out[b, h] = softmax_j(scale q_h . K_j) V,  j < used[b].
//
// The KV stream bounds it (4 D bytes a position and KV head for 4 D operations of each
// of its query heads), so everything serves that. A workgroup takes tiles of 32
// positions of one row and KV head, each of its four waves its own, without barriers,
// with two tiles of K and V in registers on their way. A tile is two halves of 16
// positions, and a page holds a multiple of 16, so a half lies in one page: its number
// is a scalar load two tiles ahead, and the lanes' offsets from the half's first
// position are constants. Every KV byte is read once, straight into MFMA operands.
//
// us per launch in a graph, 24 query heads over 8 of D = 64, random pages of 64: 128 rows
// of 1024 to 4095 positions 106.5 (6.3 TB/s of 6.9 that a bare read of such tiles
// reaches), 101.3 fused and in an order (6.6 TB/s); 64 rows of 1025 to 1279 26.1 (5.8),
// fused the same; 32 rows of 8191 to 32768 203 (6.6); 8 such rows of D = 128 106.5 (6.3);
// one row of 509 5.6 (launch, three latencies, the merge). Pages of 16 cost 1%.
//
// Scores: S = K . q^T with v_mfma_f32_16x16x32_bf16, A the 16 positions of a half
// (lane l: position l % 16, 16 bytes of channels), B the query heads of the KV head
// (column l % 16; columns past the G heads are zero). Lane l then holds positions
// 4 (l / 16) .. + 3 of both halves for query head l % 16. Loaded in that layout, an
// instruction touches 16 lines and takes half of each. K is loaded in whole lines of
// eight positions instead, and lanes 8 apart swap (24 vector instructions a tile of D
// = 64): 128 ragged rows 112.4 -> 106.5 us, bare reads of such tiles 105.1 -> 96.9.
//
// P.V: O^T = V^T . P^T. The sum over positions may take them in any order that both
// operands share, so a lane's eight probabilities are its B operand as they stand: k
// index 8 g + i is position 4 g + i of half 0, and 8 g + 4 + i that of half 1. A is
// V transposed: lane l loads channels D/16 (l % 16) .. of those eight positions
// (8 or 16 bytes each, rows of one position contiguous over 16 lanes) and pairs
// them per channel with v_perm, 2 instructions a position and 64 bytes. A row of
// the result is then a channel of the same 16-fold stride, and the lane's
// accumulators are D/4 consecutive channels.
//
// The running maximum is a column's own reference, kept kAbove over the score that
// set it and moved only when a score passes it, so nothing crosses lanes in the
// usual tile. Waves merge through LDS, a row's workgroups by log-sum-exp in a second
// launch.
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
constexpr int kMaxQkvSplits = 8, kEarlySplits = 4;  // slices of the projection, those requested before the KV stream
constexpr int kMaxGroups = 16;

// Running maximum before any position: below every finite score, and finite, so
// exp2(kEmpty - m) and exp2(-inf - kEmpty) are 0.
constexpr float kEmpty = -3.402823466e38f;
constexpr float kAbove = 8.f;

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// Results that other workgroups add to, in slots of G query heads of a KV head: one per
// (row, split), or two per share, of a row that another share began and of one that it
// began itself.
struct Partial {
  int32_t *off;    // shares: [batch + 1] tiles before each row
  float *o;        // [slot][G][D]
  float *m, *l;    // [slot][G] maxima (log2 units) and sums of the probabilities
  float *rm, *rl;  // weighed: those of rows that one workgroup held, [batch, q_heads]
  float *s;        // weighed: scores in log2 units, [batch, q_heads, padded]
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
  int q_heads, G, max_len;
  int splits;  // workgroups that take a row's tiles in turn
  int shares;  // or equal pieces that all rows' tiles are cut into (0: not)
  float scale;
  int batch;
  int round;  // rows whose workgroups fill the CUs once
};

// Positions of a row that are looked at, and their tiles.
__device__ __forceinline__ int row_length(int used, const Shape &sh, const PagedKV &kv) {
  return max(0, min(min(used, sh.max_len), kv.width << kv.shift));
}
__device__ __forceinline__ int row_tiles(int n) { return (n + kTile - 1) / kTile; }
// Tiles of a share: all rows' tiles cut evenly, one for each wave at least.
__device__ __forceinline__ uint32_t share_tiles(uint32_t total, const Shape &sh) {
  return max((total + sh.shares - 1) / (uint32_t)sh.shares, (uint32_t)kWaves);
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

// Lanes 8 .. 15 of each 16 have from `a` what lanes 0 .. 7 want to have from `b`: swapped.
__device__ __forceinline__ void in_place(u32x4 &a, u32x4 &b) {
  constexpr int kRowRor8 = 0x128;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int x = (int)a[i], y = (int)b[i];
    a[i] = (uint32_t)__builtin_amdgcn_update_dpp(x, y, kRowRor8, 0xf, 0xc, false);
    b[i] = (uint32_t)__builtin_amdgcn_update_dpp(y, x, kRowRor8, 0xf, 0x3, false);
  }
}

// Bytes of LDS before the scores: the merge of the waves and the fused prologue use the
// same ones in turn; the heads' factors behind them.
// Tiles whose scores a wave stores together; its ring takes 8 KB at most. (Eight tiles for
// every G: 135 us against 136 at 8 heads a KV head, 159 and 158 at 16.)
__host__ __device__ constexpr int ring_tiles(int G) { return G <= 4 ? 8 : 4; }
__host__ __device__ constexpr int lds_bytes(int D, int G, bool fused) {
  const int merge = kWaves * G * (D + 2) * 4, rot = fused ? (G + 2) * D * (2 + 4) : 0;
  return ((merge > rot ? merge : rot) + 2 * G * 4 + 15) / 16 * 16;
}

// What a launch reads and writes.
struct Args {
  const bf16 *q;
  int64_t qs0, qs1;
  PagedKV kv;
  const int32_t *table, *used;
  Shape sh;
  Partial part;
  QkvIn in;
  const float *before;
  float *after;
  bf16 *out;
  int out_mb;
};

// Weights: none; scores to the workspace, for a launch of their own; or scores in LDS
// and the weights added here, where a workgroup holds the row (64 rows of 1025 to 1279
// positions, 24 query heads over 8: 36.0 us by way of the workspace, 29.2 in LDS; now 27.1).
enum Weigh { kNone, kScores, kHeld };

__device__ __forceinline__ int64_t out_index(const Args &a, int64_t b, int hq, int c, int dim) {
  return a.out_mb ? frag_offset_rows(b, (int64_t)hq * dim + c, a.out_mb) : (b * a.sh.q_heads + hq) * dim + c;
}

// Row b, which holds `held` positions, n of them looked at, for KV head h: tiles lo to
// hi - 1, of each `stride` the first kWaves. The row's result where that is all of it
// (whole), else a partial one in `slot`. Every thread of the workgroup calls it.
template <int D, bool kFused, int kWeigh>
__device__ __forceinline__ void attend(const Args &a, const bf16 *__restrict__ q, const int32_t *__restrict__ table,
                                       int64_t b, int h, int held, int n, int lo, int hi, int stride, bool whole,
                                       int64_t slot, char *smem) {
  constexpr int kSteps = D / 32, kCh = D / 16;  // k steps of a score; channels a lane takes of a V row
  const PagedKV &kv = a.kv;
  const Shape &sh = a.sh;
  const QkvIn &in = a.in;
  const Partial &part = a.part;
  // Opaque, so that what follows from it is not kept in registers from row to row.
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));
  const int lane = tid % kWave, wave = scalar(tid / kWave);
  const int r = lane & 15, g = lane >> 4;
  const int G = sh.G;

  // Fused: loads of the partials first, so that nothing of the KV stream stands before them.
  const int ncols = (sh.q_heads + 2 * kv.heads) * D;
  const int stages = (G + 2) * (D / 4);  // threads' work staging 4 channels each
  f32x4 pv[kEarlySplits];
  auto source = [&](int t) {
    const int hs = t / (D / 4), c4 = t % (D / 4) * 4;
    const int head = hs < G ? h * G + hs : (hs == G ? sh.q_heads + h : sh.q_heads + kv.heads + h);
    return in.part + b * ncols + (int64_t)head * D + c4;
  };
  // and the angles of pair tid % (D / 2), the pair that the thread turns.
  constexpr int kPairs = D / 2;
  static_assert(kThreads % kPairs == 0, "a thread turns one pair of every head it takes");
  const int pair = tid % kPairs, half = in.rot.rotary / 2;
  bool in_table = false, writes = false;
  float turn_c = 1.f, turn_s = 0.f;
  u32x4 qw[kSteps];
  if constexpr (kFused) {
    if (tid < stages) {
      const float *src = source(tid);
#pragma unroll
      for (int s = 0; s < kEarlySplits; ++s)
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
      qw[s] = r < G ? *reinterpret_cast<const u32x4 *>(q + b * a.qs0 + (int64_t)(h * G + r) * a.qs1 + 32 * s + 8 * g)
                    : u32x4{0, 0, 0, 0};
  }

  const int first = lo + wave, tiles = row_tiles(n);  // this wave's tiles: first, first + stride, ...
  const int32_t *row_table = table + b * kv.width;
  // K is loaded in whole lines, eight positions an instruction, and put in place by
  // in_place(): lane (r, g) loads 16 bytes of positions r % 8 and r % 8 + 8.
  const uint32_t k_off = (uint32_t)(r % 8 * D + (r / 8 * 4 + g) * 8) * 2, v_off = (uint32_t)(4 * g * D + r * kCh) * 2;
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
  // In bounds whatever the table holds: a page that does not exist, and a tile past the
  // end, are read from page 0. So the table's words need not wait for the row's length.
  auto load = [&](Kv<D> &x, const Ids &ids, int tile) {
    const int j = tile * kTile;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int id = ids.id[t];
      x.ok[t] = (uint32_t)id < (uint32_t)kv.pages;
      const int64_t from =
          ((((int64_t)(x.ok[t] && tile < hi ? id : 0) * kv.heads + h) << kv.shift) + ((j + 16 * t) & page_mask)) * D;
      const char *kb = reinterpret_cast<const char *>(kv.k + from), *vb = reinterpret_cast<const char *>(kv.v + from);
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
        x.k[t][s] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(kb + k_off + (s % 2 * 8 * D + s / 2 * 64) * 2));
#pragma unroll
      for (int i = 0; i < 4; ++i)
        x.v[t][i] = __builtin_nontemporal_load(reinterpret_cast<const typename Kv<D>::V *>(vb + v_off + 2 * D * i));
    }
  };
  // The first two tiles are on their way before anything else is waited for, without a
  // branch: loads under one would make the wait counts fall back to waiting for all.
  Kv<D> xa, xb;
  const Ids ia = ids_of(first), ib = ids_of(first + stride);
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
    if (tid < stages) {
      f32x4 sum = pv[0];
#pragma unroll
      for (int s = 1; s < kEarlySplits; ++s)
        if (s < in.splits) sum += pv[s];
      for (int s = kEarlySplits; s < in.splits; ++s)
        sum += *reinterpret_cast<const f32x4 *>(source(tid) + (int64_t)s * sh.batch * ncols);
      stage(tid, sum);
    }
    for (int t = tid + kThreads; t < stages; t += kThreads) {
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
    for (int hs = tid / kPairs; hs < G + 2; hs += kThreads / kPairs) {
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
    if (writes && n > 0 && held == n && (tiles - 1 - lo) % stride < kWaves && hi == tiles) {
      const int id = constant(row_table + (last >> kv.shift));
      own = (uint32_t)id < (uint32_t)kv.pages;
      new_cell = ((((int64_t)(own ? id : 0) * kv.heads + h) << kv.shift) + (last & page_mask)) * D;
    }
  }

  // kHeld: factors of the query heads, and the row's scores
  float *sm_f = reinterpret_cast<float *>(smem + lds_bytes(D, G, kFused)) - 2 * G;
  float *sm_s = sm_f + 2 * G;
  const int sm_padded = (sh.max_len + kTile - 1) / kTile * kTile;
  // kScores: a wave's scores of its last tiles, stored together, whole lines of one head by
  // eight lanes. Loads and stores return in the order they were issued, so a store behind
  // every tile holds the stream up: 64 rows of 500 to 8000 positions, 3 query heads per KV
  // head, 137 us with one behind every tile, 133 in this way (K in half lines; now 119).
  const int ring = ring_tiles(G);
  float *sm_ring = sm_f + 2 * G + wave * ring * G * kTile;
  int ringed = 0;
  auto store_scores = [&](int end) {  // of the tiles before `end`
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // other lanes wrote what this one reads
    // 8 lanes a tile and head, four positions each
    const int at = lane / 8 % ring, c = lane % 8 * 4;
    const int64_t to = (int64_t)(end - (ringed - at) * stride) * kTile + c;
    for (int gh = lane / 8 / ring; gh < G; gh += 8 / ring)
      if (at < ringed)
        *reinterpret_cast<f32x4 *>(part.s + (b * sh.q_heads + h * G + gh) * part.padded + to) =
            *reinterpret_cast<const f32x4 *>(sm_ring + (at * G + gh) * kTile + c);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    ringed = 0;
  };
  const float sl2 = sh.scale * 1.4426950408889634f;
  float m = kEmpty, l = 0.f;  // l: of the lane's own positions
  f32x4 acc[kCh];
#pragma unroll
  for (int c = 0; c < kCh; ++c) acc[c] = f32x4{0.f, 0.f, 0.f, 0.f};

  auto compute = [&](Kv<D> &x, int tile) {
    const int left = n - tile * kTile;  // positions of the row from this tile on
    const bool edge = left < kTile || (kFused && own && tile == tiles - 1) || !x.ok[0] || !x.ok[1];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int s = 0; s < kSteps; s += 2) in_place(x.k[t][s], x.k[t][s + 1]);
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
    if constexpr (kWeigh != kNone) {
      if (r < G) {
        float *to = kWeigh == kHeld ? sm_s + r * sm_padded + tile * kTile : sm_ring + (ringed * G + r) * kTile;
#pragma unroll
        for (int t = 0; t < 2; ++t)
          *reinterpret_cast<f32x4 *>(to + 4 * g + 16 * t) = f32x4{sc[t][0], sc[t][1], sc[t][2], sc[t][3]};
      }
      ++ringed;
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
      l *= f;
#pragma unroll
      for (int cb = 0; cb < kCh; ++cb) acc[cb] *= f;
    }
    // Probabilities for the matrix cores in two bf16 parts, cut and rest: with one, rounded
    // (2^-9 of each off), results were off by 2.2e-3 (relative, RMS), with two by 1.7e-3, the
    // output's own rounding, in the same time. The rest is taken 2^-18 of the whole larger,
    // so that for probabilities of 2^-108 and more (of the running maximum's) it is a normal
    // number above 0: 0 times an infinity in V is no number, which an infinity attended by a
    // smaller one may give.
    u32x4 p, rest;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float p0 = __builtin_amdgcn_exp2f(sc[t][2 * i] - m), p1 = __builtin_amdgcn_exp2f(sc[t][2 * i + 1] - m);
        l += p0;
        l += p1;
        const uint32_t b0 = __float_as_uint(p0), b1 = __float_as_uint(p1);
        p[2 * t + i] = __builtin_amdgcn_perm(b1, b0, 0x07060302u);
        rest[2 * t + i] = pack_bf16_nc(__builtin_fmaf(p0, 1.f + 0x1p-18f, -hi_f32(b0)),
                                       __builtin_fmaf(p1, 1.f + 0x1p-18f, -hi_f32(b1)));
      }
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
      acc[cb] = mfma16x16x32(vt, rest, acc[cb]);
    }
  };

  // Tiles in pairs while there is one to load for the first of the two; the second may
  // be past the end, once.
  int tile = first;
  for (; tile + 2 * stride < hi; tile += 2 * stride) {
    compute(xa, tile);
    load(xa, na, tile + 2 * stride);
    compute(xb, tile + stride);
    load(xb, nb, tile + 3 * stride);
    na = ids_of(tile + 4 * stride);
    nb = ids_of(tile + 5 * stride);
    if constexpr (kWeigh == kScores) {
      if (ringed == ring) store_scores(tile + 2 * stride);
    }
  }
  if (tile < hi) compute(xa, tile);
  if (tile + stride < hi) compute(xb, tile + stride);
  if constexpr (kWeigh == kScores) store_scores(tile + (tile < hi) * stride + (tile + stride < hi) * stride);

  if constexpr (kFused) {
    // Stored behind the stream, which does not wait for it.
    if (own && tid < D / 4) {
      const int side = tid / (D / 8), c = tid % (D / 8) * 8;
      *reinterpret_cast<u32x4 *>((side ? kv.v : kv.k) + new_cell + c) =
          *reinterpret_cast<const u32x4 *>(&sm_rot[G + side][c]);
    }
    __syncthreads();  // sm_rot is done with
  }
  l += xor_lanes<16>(l);
  l += xor_lanes<32>(l);
  // Waves merge: [wave][G][D] accumulators, then [wave][G] of m and l.
  float *sm_o = reinterpret_cast<float *>(smem);
  float *sm_m = sm_o + kWaves * G * D, *sm_l = sm_m + kWaves * G;
  if (r < G) {
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
      for (int cb = 0; cb < kCh; cb += 4)
        *reinterpret_cast<f32x4 *>(sm_o + (wave * G + r) * D + (4 * g + x) * kCh + cb) =
            f32x4{acc[cb][x], acc[cb + 1][x], acc[cb + 2][x], acc[cb + 3][x]};
    if (g == 0) {
      sm_m[wave * G + r] = m;
      sm_l[wave * G + r] = l;
    }
  }
  __syncthreads();
  for (int t = tid; t < G * D; t += kThreads) {
    const int gh = t / D, c = t % D;
    float mx = sm_m[gh];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) mx = fmaxf(mx, sm_m[w * G + gh]);
    float lsum = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float f = __builtin_amdgcn_exp2f(sm_m[w * G + gh] - mx);
      lsum += sm_l[w * G + gh] * f;
      o += sm_o[(w * G + gh) * D + c] * f;
    }
    const int hq = h * G + gh;
    if (whole) {
      a.out[out_index(a, b, hq, c, D)] = (bf16)f32_to_bf16(lsum == 0.f ? 0.f : o / lsum);
      if constexpr (kWeigh == kScores) {
        if (c == 0) {
          part.rm[b * sh.q_heads + hq] = mx;
          part.rl[b * sh.q_heads + hq] = lsum;
        }
      }
      if constexpr (kWeigh == kHeld) {
        if (c == 0) {
          sm_f[gh] = mx;
          sm_f[G + gh] = lsum == 0.f ? 0.f : 1.f / lsum;
        }
      }
    } else {
      const int64_t at = slot * G + gh;
      part.o[at * D + c] = o;
      if (c == 0) {
        part.m[at] = mx;
        part.l[at] = lsum;
      }
    }
  }
  if constexpr (kWeigh == kHeld) {
    __syncthreads();
    // Four positions a thread; a row's positions in the weights are a multiple of 16.
    const int64_t row = (b * kv.heads + h) * ((int64_t)kv.width << kv.shift);
    for (int j = 4 * tid; j < n; j += 4 * kThreads) {
      const f32x4 old = *reinterpret_cast<const f32x4 *>(a.before + row + j);
      float w[4] = {0.f, 0.f, 0.f, 0.f};
      for (int gh = 0; gh < G; ++gh) {
        const f32x4 sc = *reinterpret_cast<const f32x4 *>(sm_s + gh * sm_padded + j);
        const float mg = sm_f[gh], f = sm_f[G + gh];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] += __builtin_amdgcn_exp2f(sc[i] - mg) * f;
      }
      if (j + 4 <= n) {
        *reinterpret_cast<f32x4 *>(a.after + row + j) = f32x4{old[0] + w[0], old[1] + w[1], old[2] + w[2], old[3] + w[3]};
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (j + i < n) a.after[row + j + i] = old[i] + w[i];
      }
    }
  }
}

// grid (kv heads, splits, rows): a row's tiles go to the waves of all its splits in
// turn, so that nothing but the end of the loop waits for its length. Or grid (kv
// heads, shares): the tiles of all rows, one row after the other, are cut evenly, so
// that every workgroup streams as many bytes whatever the rows' lengths. A CU alone
// reads some 35 GB/s, so the rate of the whole falls with its emptiest CU; a workgroup
// adds up the rows' tiles itself.
// Registers: four waves per SIMD where splits give a CU four workgroups (D = 64). With
// scores to store that would spill (64 rows of 500 to 8000 positions, 3 query heads per KV
// head, when three took 133 us: 145), and shares give a CU two.
template <int D, bool kFused, int kWeigh, bool kShares>
__global__ void __launch_bounds__(kThreads, D == 128 || kShares ? 2 : kWeigh == kScores ? 3 : 4)
decode_paged_kernel(const bf16 *__restrict__ q, const int32_t *__restrict__ table, Args a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int h = blockIdx.x;
  if constexpr (!kShares) {
    const int split = blockIdx.y, splits = a.sh.splits;
    // An order's rows go to the CUs forth and back: one whose first row is a round's longest
    // has the next round's shortest (128 rows of 1024 to 4095 positions, longest first:
    // 105.0 us without, 101.1 so).
    int64_t b = blockIdx.z;
    if (kFused && a.in.order) {
      const int z = blockIdx.z, from = z / a.sh.round * a.sh.round, to = min(from + a.sh.round, a.sh.batch);
      b = constant(a.in.order + (z / a.sh.round % 2 ? from + to - 1 - z : z));
    }
    const int held = constant(a.used + b), n = row_length(held, a.sh, a.kv), tiles = row_tiles(n);
    if (splits > 1 && split * kWaves >= tiles) return;
    attend<D, kFused, kWeigh>(a, q, table, b, h, held, n, split * kWaves, tiles, splits * kWaves,
                              splits == 1 || tiles <= kWaves, (b * splits + split) * a.kv.heads + h, smem);
  } else {
    const int lane = threadIdx.x % kWave, batch = a.sh.batch;
    uint32_t total = 0;
    for (int b = lane; b < batch; b += kWave) total += row_tiles(row_length(a.used[b], a.sh, a.kv));
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) total += shfl_xor(total, d);
    total = scalar(total);
    const uint32_t share = share_tiles(total, a.sh);
    const uint32_t start = min(blockIdx.y * share, total), end = min(start + share, total);
    const bool writer = h == 0 && blockIdx.y == 0 && threadIdx.x < kWave;
    uint32_t before = 0, row_off = 0;
    int row = batch;  // the row that holds tile `start`, and the tiles before it
    for (int b0 = 0; b0 < batch && (row == batch || writer); b0 += kWave) {
      const int b = b0 + lane;
      const uint32_t mine = b < batch ? row_tiles(row_length(a.used[b], a.sh, a.kv)) : 0;
      uint32_t upto = mine;
#pragma unroll
      for (int d = 1; d < kWave; d *= 2) {
        const uint32_t y = __shfl_up(upto, d, kWave);
        upto += lane >= d ? y : 0;
      }
      if (writer && b < batch) a.part.off[b] = (int)(before + upto - mine);
      const uint64_t there = __ballot(start < before + upto);
      if (row == batch && there) {
        const int at = __builtin_ctzll(there);
        row = b0 + at;
        row_off = before + __shfl(upto - mine, at, kWave);
      }
      before += __shfl(upto, kWave - 1, kWave);
    }
    if (writer && lane == 0) a.part.off[batch] = (int)total;
    if (start >= end) return;  // more shares than the rows have tiles for
    row = scalar(row);
    row_off = scalar(row_off);
    while (row_off < end) {  // uniform: every wave has the same numbers
      const int held = constant(a.used + row), n = row_length(held, a.sh, a.kv), tiles = row_tiles(n);
      if (tiles) {
        const int lo = row_off < start ? (int)(start - row_off) : 0, hi = (int)min((uint32_t)tiles, end - row_off);
        attend<D, kFused, kWeigh>(a, q, table, row, h, held, n, lo, hi, kWaves, lo == 0 && hi == tiles,
                                  ((int64_t)blockIdx.y * a.kv.heads + h) * 2 + (lo ? 0 : 1), smem);
        __syncthreads();  // the next row takes the same LDS
      }
      row_off += tiles;
      ++row;
    }
  }
}

// The partial results of a row: `count` of them, 0 of an empty row, 1 where a workgroup
// held it all and wrote its result.
struct Pieces {
  int n, count;
  int64_t first;  // shares: the first one; splits: b * splits
  bool shares;
};
__device__ __forceinline__ Pieces pieces_of(const Args &a, int64_t b) {
  Pieces x;
  x.n = row_length(a.used[b], a.sh, a.kv);
  x.shares = a.sh.shares > 0;
  if (x.shares) {
    const uint32_t at = a.part.off[b], next = a.part.off[b + 1], share = share_tiles(a.part.off[a.sh.batch], a.sh);
    x.first = at / share;
    x.count = next > at ? (int)((next - 1) / share - at / share) + 1 : 0;
  } else {
    x.first = b * a.sh.splits;
    x.count = min(a.sh.splits, (row_tiles(x.n) + kWaves - 1) / kWaves);
  }
  return x;
}
// Query head gh of KV head h in the row's i-th piece (its first share began the row).
__device__ __forceinline__ int64_t slot_of(const Args &a, const Pieces &x, int i, int h, int gh) {
  const int64_t at = (x.first + i) * a.kv.heads + h;
  return (x.shares ? 2 * at + (i ? 0 : 1) : at) * a.sh.G + gh;
}

// Channel c of a row's result from its pieces, by log-sum-exp; the results of kBatch
// pieces are requested together, of the first `slots` ones.
constexpr int kBatch = 8;
template <int D>
__device__ __forceinline__ float joined(const Args &a, const Pieces &x, int slots, int h, int gh, int c) {
  const Partial &part = a.part;
  float mx = kEmpty, lsum = 0.f, o = 0.f;
  for (int s0 = 0; s0 < x.count; s0 += kBatch) {
    float ms[kBatch], ls[kBatch], os[kBatch], to = mx;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int64_t at = slot_of(a, x, min(s0 + i, slots - 1), h, gh);
      ms[i] = part.m[at];
      ls[i] = part.l[at];
      os[i] = part.o[at * D + c];
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) to = fmaxf(to, s0 + i < x.count ? ms[i] : kEmpty);
    const float f0 = __builtin_amdgcn_exp2f(mx - to);
    lsum *= f0;
    o *= f0;
    mx = to;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const bool live = s0 + i < x.count;
      const float f = live ? __builtin_amdgcn_exp2f(ms[i] - mx) : 0.f;
      lsum += live ? ls[i] * f : 0.f;
      o += live ? os[i] * f : 0.f;
    }
  }
  return lsum == 0.f ? 0.f : o / lsum;
}

// Rows in several pieces: their results; rows that hold nothing: zeros. grid (groups of
// query heads, batch), one thread per channel.
constexpr int kCombineHeads = 2;
template <int D>
__global__ void __launch_bounds__(kCombineHeads *D)
decode_paged_combine_kernel(Args a) {
  const int hq = blockIdx.x * kCombineHeads + threadIdx.x / D;
  const int64_t b = blockIdx.y;
  const Pieces x = pieces_of(a, b);
  if (hq >= a.sh.q_heads || x.count == 1) return;
  const int c = threadIdx.x % D;
  // The first results need not wait for the row's length: every split has a slot, and
  // what a split past the row's end has there is not looked at.
  const float o = joined<D>(a, x, x.shares ? x.count : a.sh.splits, hq / a.sh.G, hq % a.sh.G, c);
  a.out[out_index(a, b, hq, c, D)] = (bf16)f32_to_bf16(o);
}

// after[b, h, j] = before[b, h, j] + sum over the KV head's query heads of their
// probability of position j, j < the row's length. A thread four positions. The first
// workgroups of a (row, KV head) join the pieces' results, as the launch above.
// Bound by the scores' way to memory and back (24 bytes a position and KV head of three
// query heads, beside 256 of K and V) and, in small calls, by its launch: 64 rows of 500
// to 8000 positions in shares 119 us with weights and 89.5 without, 3 rows to 4001 11.2 and
// 10.6, 3 rows to 6157 with 16 query heads a KV head and D = 128 24.6 and 19.4. There the
// first workgroup of a (row, KV head) joined all its pieces before: 43.4.
constexpr int kWeighThreads = 256, kWeighSpan = 4 * kWeighThreads;
template <int D>
__global__ void __launch_bounds__(kWeighThreads)
weigh_kernel(Args a) {
  const int h = blockIdx.y, G = a.sh.G, tid = threadIdx.x;
  const int64_t b = blockIdx.z;
  const Partial &part = a.part;
  const int joins = (G * D + kWeighThreads - 1) / kWeighThreads, span = (int)blockIdx.x - joins;
  if (span < 0) {
    const Pieces x = pieces_of(a, b);
    const int t = blockIdx.x * kWeighThreads + tid, gh = t / D, c = t % D;
    if (x.count == 1 || gh >= G) return;
    a.out[out_index(a, b, h * G + gh, c, D)] = (bf16)f32_to_bf16(joined<D>(a, x, x.count, h, gh, c));
    return;
  }
  const int n = row_length(a.used[b], a.sh, a.kv), j = span * kWeighSpan + tid * 4;
  if (span * kWeighSpan >= n) return;
  // The scores and weights of this thread's positions are on their way while the
  // heads' sums are joined. The buffers hold a multiple of 16 positions a row.
  const float *sc = part.s + (b * a.sh.q_heads + h * G) * part.padded + j;
  const int64_t at = (b * a.kv.heads + h) * ((int64_t)a.kv.width << a.kv.shift) + j;
  f32x4 s[kMaxGroups], old{0.f, 0.f, 0.f, 0.f};
  if (j < n) {
#pragma unroll
    for (int gh = 0; gh < kMaxGroups; ++gh)
      if (gh < G) s[gh] = *reinterpret_cast<const f32x4 *>(sc + gh * part.padded);
    old = *reinterpret_cast<const f32x4 *>(a.before + at);
  }
  // Every head by 16 lanes.
  __shared__ float sm_m[kMaxGroups], sm_f[kMaxGroups];
  const Pieces x = pieces_of(a, b);
  constexpr int kLanes = kWeighThreads / kMaxGroups;
  const int gh = tid / kLanes, lane = tid % kLanes;
  float mx = kEmpty, l = 0.f;
  if (gh < G) {
    if (x.count == 1) {
      mx = part.rm[b * a.sh.q_heads + h * G + gh];
      l = lane == 0 ? part.rl[b * a.sh.q_heads + h * G + gh] : 0.f;
    } else {
      for (int i = lane; i < x.count; i += kLanes) {
        const int64_t slot = slot_of(a, x, i, h, gh);
        const float m = part.m[slot], more = part.l[slot], to = fmaxf(mx, m);
        l = l * __builtin_amdgcn_exp2f(mx - to) + more * __builtin_amdgcn_exp2f(m - to);
        mx = to;
      }
    }
  }
  float to = mx;
#pragma unroll
  for (int d = 1; d < kLanes; d *= 2) to = fmaxf(to, shfl_xor(to, d));
  l *= __builtin_amdgcn_exp2f(mx - to);
#pragma unroll
  for (int d = 1; d < kLanes; d *= 2) l += shfl_xor(l, d);
  if (lane == 0) {
    sm_m[gh] = to;
    sm_f[gh] = l == 0.f ? 0.f : 1.f / l;
  }
  __syncthreads();
  if (j >= n) return;
  float w[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int gh = 0; gh < kMaxGroups; ++gh) {
    if (gh < G) {
      const float m = sm_m[gh], f = sm_f[gh];
#pragma unroll
      for (int y = 0; y < 4; ++y) w[y] += __builtin_amdgcn_exp2f(s[gh][y] - m) * f;
    }
  }
  if (j + 4 <= n) {
    *reinterpret_cast<f32x4 *>(a.after + at) = f32x4{old[0] + w[0], old[1] + w[1], old[2] + w[2], old[3] + w[3]};
  } else {
#pragma unroll
    for (int y = 0; y < 4; ++y)
      if (j + y < n) a.after[at + y] = old[y] + w[y];
  }
}

struct Call {
  int64_t batch, q_heads, kv_heads, head_dim, width, pages, page, max_len, num_splits, num_shares;
};

int64_t padded_scores(int64_t max_len) { return align_up(max_len, kTile); }

// Scores that a workgroup keeps: with the merge they fit a CU's 160 KB of LDS, though one
// workgroup then has it to itself. us with weights, in LDS and by way of memory (in shares,
// where that is faster), 8 KV heads: 64 rows of 1025 to 1279 positions, 8 query heads each
// (40 KB) 28.1 and 44.3, 16 (80 KB) 35.0 and 48.6; 64 rows of 1024 to 4000, 3 query heads
// (47 KB) 62.0 and 72.9; 128 such rows, 6 query heads (94 KB) 119 and 154; 64 rows of 500 to
// 8000, 3 (94 KB) 106 and 119; 32 rows of 500 to 9000, 3 (106 KB) 65.5 and 69.0.
constexpr int64_t kHeldBytes = 120 << 10;
static_assert(kHeldBytes + lds_bytes(128, kMaxGroups, true) <= 160 << 10, "the LDS of a CU");
bool scores_held(int64_t groups, int64_t max_len) { return groups * padded_scores(max_len) * 4 <= kHeldBytes; }

// Weights added by the workgroup that holds the row.
bool weighs_held(int64_t groups, int64_t max_len, int64_t splits, int64_t shares) {
  return splits == 1 && !shares && scores_held(groups, max_len);
}

int64_t slot_count(int64_t batch, int64_t kv_heads, int64_t splits, int64_t shares) {
  return shares ? shares * kv_heads * 2 : splits > 1 ? batch * splits * kv_heads : 0;
}

int64_t workspace_bytes(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t max_len,
                        int64_t splits, int64_t shares, bool weighed) {
  const int64_t n = slot_count(batch, kv_heads, splits, shares) * (q_heads / kv_heads);
  const bool scores = weighed && !weighs_held(q_heads / kv_heads, max_len, splits, shares);
  return (shares ? align_up((batch + 1) * 4, 256) : 0) + align_up(n * head_dim * 4, 256) + 2 * align_up(n * 4, 256) +
         (scores ? 2 * align_up(batch * q_heads * 4, 256) + batch * q_heads * padded_scores(max_len) * 4 : 0);
}

bool pieces_ok(int64_t splits, int64_t shares) {
  return splits >= 1 && splits <= 1024 && shares >= 0 && shares <= 65535 && (splits == 1 || shares == 0);
}

// Argument checks of both entry points; *run false where nothing is to launch.
int check_call(const Call &c, bool *run) {
  *run = false;
  LM_REQUIRE(c.batch >= 0 && c.q_heads > 0 && c.kv_heads > 0 && c.q_heads % c.kv_heads == 0 && c.max_len > 0 &&
             pieces_ok(c.num_splits, c.num_shares) && c.max_len < ((int64_t)1 << 30) && c.batch <= 65535 &&
             c.kv_heads <= 65535);
  const int status = paged_args_ok(c.width, c.pages, c.page, c.head_dim);
  if (status != LM_OK) return status;
  if (c.q_heads / c.kv_heads > kMaxGroups) return LM_EUNSUPPORTED;
  // tiles of all rows are counted in 32 bits
  LM_REQUIRE(c.batch <= ((int64_t)1 << 31) / cdiv(c.max_len, kTile));
  *run = c.batch > 0;
  return LM_OK;
}

template <int D, bool kFused, int kWeigh, bool kShares>
int launch_sized(const Call &c, const Args &a, hipStream_t s) {
  // KV heads fastest: workgroups go to the XCDs in turn, so that each XCD has some of
  // every row.
  const dim3 grid = kShares ? dim3((unsigned)c.kv_heads, (unsigned)a.sh.shares)
                            : dim3((unsigned)c.kv_heads, (unsigned)a.sh.splits, (unsigned)c.batch);
  const int64_t lds = lds_bytes(D, a.sh.G, kFused) + (kWeigh == kHeld     ? a.sh.G * padded_scores(a.sh.max_len) * 4
                                                      : kWeigh == kScores ? kWaves * ring_tiles(a.sh.G) * a.sh.G * kTile * 4
                                                                          : 0);
  decode_paged_kernel<D, kFused, kWeigh, kShares><<<grid, kThreads, lds, s>>>(a.q, a.table, a);
  LM_CHECK_LAUNCH();
  if (kWeigh == kNone && (kShares || a.sh.splits > 1)) {
    decode_paged_combine_kernel<D><<<dim3((unsigned)cdiv(c.q_heads, kCombineHeads), (unsigned)c.batch),
                                     kCombineHeads * D, 0, s>>>(a);
    LM_CHECK_LAUNCH();
  }
  if (kWeigh == kScores) {
    const int64_t joins = cdiv(a.sh.G * D, kWeighThreads);
    weigh_kernel<D><<<dim3((unsigned)(joins + cdiv(a.sh.max_len, kWeighSpan)), (unsigned)c.kv_heads, (unsigned)c.batch),
                      kWeighThreads, 0, s>>>(a);
    LM_CHECK_LAUNCH();
  }
  return LM_OK;
}

int launch_decode_paged(const Call &c, Args a, void *workspace, int64_t workspace_bytes_, void *stream) {
  LM_REQUIRE(aligned16(a.kv.k) && aligned16(a.kv.v) && (a.before == nullptr) == (a.after == nullptr) &&
             aligned16(a.before) && aligned16(a.after));
  LM_REQUIRE(in_place_or_apart(a.before, a.after, c.batch * c.kv_heads * c.width * c.page * 4));
  const bool weighed = a.after != nullptr;
  const int64_t G = c.q_heads / c.kv_heads;
  const bool held = weighed && weighs_held(G, c.max_len, c.num_splits, c.num_shares);
  const int64_t need = workspace_bytes(c.batch, c.q_heads, c.kv_heads, c.head_dim, c.max_len, c.num_splits,
                                       c.num_shares, weighed);
  if (need > 0 && (!workspace || workspace_bytes_ < need)) return LM_EWORKSPACE;
  LM_REQUIRE(need == 0 || aligned16(workspace));
  // No row is longer than the table.
  const int64_t room = c.width * c.page, longest = c.max_len < room ? c.max_len : room;
  a.sh.q_heads = (int)c.q_heads;
  a.sh.G = (int)G;
  a.sh.max_len = (int)longest;
  a.sh.splits = (int)c.num_splits;
  a.sh.shares = (int)c.num_shares;
  a.sh.batch = (int)c.batch;
  a.sh.round = (int)(c.kv_heads < 256 ? 256 / c.kv_heads : 1);
  a.kv.pages = c.pages;
  a.kv.width = (int)c.width;
  a.kv.shift = page_shift(c.page);
  a.kv.heads = (int)c.kv_heads;
  a.part = Partial{};
  a.part.padded = padded_scores(c.max_len);
  char *w = static_cast<char *>(workspace);
  auto take = [&](int64_t count) {
    char *at = w;
    w += align_up(count * 4, 256);
    return reinterpret_cast<float *>(at);
  };
  const int64_t n = slot_count(c.batch, c.kv_heads, c.num_splits, c.num_shares) * G;
  if (c.num_shares) a.part.off = reinterpret_cast<int32_t *>(take(c.batch + 1));
  a.part.o = take(n * c.head_dim);
  a.part.m = take(n);
  a.part.l = take(n);
  if (weighed && !held) {
    a.part.rm = take(c.batch * c.q_heads);
    a.part.rl = take(c.batch * c.q_heads);
    a.part.s = take(c.batch * c.q_heads * a.part.padded);
  }
  hipStream_t s = (hipStream_t)stream;
  auto run = [&](auto dim, auto fused) {
    constexpr int D = decltype(dim)::value;
    constexpr bool kFused = decltype(fused)::value;
    if (held) return launch_sized<D, kFused, kHeld, false>(c, a, s);
    if constexpr (!kFused) {
      if (c.num_shares)
        return weighed ? launch_sized<D, false, kScores, true>(c, a, s) : launch_sized<D, false, kNone, true>(c, a, s);
    }
    return weighed ? launch_sized<D, kFused, kScores, false>(c, a, s) : launch_sized<D, kFused, kNone, false>(c, a, s);
  };
  auto sized = [&](auto dim) { return a.in.part ? run(dim, std::true_type{}) : run(dim, std::false_type{}); };
  return c.head_dim == 64 ? sized(std::integral_constant<int, 64>{}) : sized(std::integral_constant<int, 128>{});
}

}  // namespace
}  // namespace lm

using namespace lm;

extern "C" int lm_flash_decode_paged_workspace_size(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                                                    int64_t max_len, int64_t num_splits, int64_t num_shares,
                                                    int weighed, int64_t *bytes) {
  LM_REQUIRE(bytes && batch >= 0 && q_heads > 0 && kv_heads > 0 && q_heads % kv_heads == 0 && max_len > 0 &&
             pieces_ok(num_splits, num_shares));
  if (head_dim != 64 && head_dim != 128) return LM_EUNSUPPORTED;
  *bytes = workspace_bytes(batch, q_heads, kv_heads, head_dim, max_len, num_splits, num_shares, weighed != 0);
  return LM_OK;
}

extern "C" int lm_flash_decode_paged(const lm_flash_decode_paged_args *args, void *stream) {
  LM_REQUIRE(args);
  const auto &x = *args;
  const Call c{x.batch, x.q_heads, x.kv_heads, x.head_dim, x.width, x.pages, x.page, x.max_len, x.num_splits, x.num_shares};
  bool run;
  const int status = check_call(c, &run);
  if (status != LM_OK || !run) return status;
  LM_REQUIRE(x.q && x.k_pages && x.v_pages && x.block_table && x.used && x.out);
  LM_REQUIRE(aligned16(x.q) && x.qs0 % 8 == 0 && x.qs1 % 8 == 0);
  Args a{};
  a.q = (const bf16 *)x.q;
  a.qs0 = x.qs0;
  a.qs1 = x.qs1;
  a.kv.k = (bf16 *)const_cast<void *>(x.k_pages);
  a.kv.v = (bf16 *)const_cast<void *>(x.v_pages);
  a.table = x.block_table;
  a.used = x.used;
  a.sh.scale = (float)x.scale;
  a.before = x.weights;
  a.after = x.weights_out;
  a.out = (bf16 *)x.out;
  return launch_decode_paged(c, a, x.workspace, x.workspace_bytes, stream);
}

extern "C" int lm_flash_decode_paged_qkv(const lm_flash_decode_paged_qkv_args *args, void *stream) {
  LM_REQUIRE(args);
  const auto &x = *args;
  const Call c{x.batch, x.q_heads, x.kv_heads, x.head_dim, x.width, x.pages, x.page, x.max_len, x.num_splits, 0};
  bool run;
  const int status = check_call(c, &run);
  if (status != LM_OK) return status;
  LM_REQUIRE(x.qkv_splits >= 1);
  if (x.qkv_splits > kMaxQkvSplits || (x.frag_out && x.batch > 128)) return LM_EUNSUPPORTED;
  if (!run) return LM_OK;
  LM_REQUIRE(x.qkv_partials && x.positions && x.k_pages && x.v_pages && x.block_table && x.used && x.out);
  LM_REQUIRE(aligned16(x.qkv_partials) && rotation_ok(x.cos_sin, x.table_len, x.rotary, x.head_dim));
  Args a{};
  a.kv.k = (bf16 *)x.k_pages;
  a.kv.v = (bf16 *)x.v_pages;
  a.table = x.block_table;
  a.used = x.used;
  a.sh.scale = (float)x.scale;
  a.in = {x.qkv_partials, (int)x.qkv_splits,
          {x.cos_sin, x.table_len, (int)x.rotary, x.table_f32 != 0, x.neox != 0}, x.positions, x.active, x.row_order};
  a.before = x.weights;
  a.after = x.weights_out;
  a.out = (bf16 *)x.out;
  a.out_mb = x.frag_out ? frag_row_blocks(x.batch) : 0;
  return launch_decode_paged(c, a, x.workspace, x.workspace_bytes, stream);
}
