// Eviction from a paged cache by weight: of a row's n = used[b] positions, per
// layer and KV head, the `recent` last ones and the heaviest of the others stay,
// `keep` in all, in their order.
//
// Selection, one workgroup per (layer, row, KV head), the row's weights in LDS. The bin of
// the keep-th heaviest by radix over the weights as ordered integers (11, 11 and 10
// bits from the top), until a bin holds few enough to rank each against all; of equal
// weights the first goes before, so there is one last that stays. Then the kept
// indices and weights are written in order, a wave a stretch of the row. Whole numbers
// throughout, so the order of the counting does not show.
//
// Move: every kept position's K and V go from the row's pages to their place in the
// target's pages, a second launch over (kept, KV head, layer and row). Out of place,
// so that pages which another row shares are left as they are and no order of the
// moves matters. Bound by the copy: 8 layers of 16 rows, 1024 positions of 8 heads of 64
// channels each (537 MB in and out) 105 us, 5.1 TB/s (a copy of 2 GiB 4.9). The selection
// of those 1024 rows of 2049 to 4095 weights, 33 MB in and out, takes 23 us: latency of
// LDS and of the passes one after the other; 128 rows of 600 to 700 6.2 us.
//
// The reference holds every position to the end (litemoe/cache.py:7-20).
#include "paged.h"

namespace lm {
namespace {

constexpr int kBins = 1 << 11;
constexpr int kCandidates = 32;          // weights of one bin that are ranked one against all
constexpr int64_t kHeldWeights = 12288;  // of a row, in LDS: with the bins less than 64 KB

// Larger floats, larger keys: -0 as 0, a NaN above every number.
__device__ __forceinline__ uint32_t key_of(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.f);
  return u ^ ((int32_t)u < 0 ? 0xffffffffu : 0x80000000u);
}
// A weight and its position as one number: heavier ones are larger, of equal ones the
// first.
__device__ __forceinline__ uint64_t order_of(uint32_t key, int j) { return (uint64_t)key << 32 | ~(uint32_t)j; }

// A value that is the same in every lane, for the scalar unit.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Sum over the lanes below this one, and over all.
__device__ __forceinline__ int wave_prefix(int v, int lane, int &total) {
  int x = v;
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const int y = __shfl_up(x, d, kWave);
    if (lane >= d) x += y;
  }
  total = __shfl(x, kWave - 1, kWave);
  return x - v;
}

// kHeld: the row's weights are read into LDS once, and may be their own output; else they
// are read from memory each time.
template <int kThreads, bool kHeld>
__global__ void __launch_bounds__(kThreads)
evict_select_kernel(const int32_t *__restrict__ used, const float *weights, int64_t capacity, int keep, int recent,
                    float *weights_out, int32_t *__restrict__ kept, int32_t *__restrict__ used_out) {
  constexpr int kWaves = kThreads / kWave, kOwn = kBins / kThreads;
  extern __shared__ __attribute__((aligned(16))) float sm_w[];
  __shared__ __attribute__((aligned(16))) int bins[kBins];
  __shared__ __attribute__((aligned(16))) uint64_t sm_candidate[kCandidates];
  __shared__ uint64_t sm_least;
  __shared__ int sm_wave[kWaves];
  __shared__ int sm_found[3];
  __shared__ int sm_candidates;
  const int h = blockIdx.x, heads = gridDim.x;
  const int64_t b = blockIdx.y, batch = gridDim.y, layer = blockIdx.z;
  const int64_t row = (layer * batch + b) * heads + h;
  const float *w = weights + row * capacity;
  float *w_out = weights_out + row * capacity;
  int32_t *to = kept + row * keep;
  const int tid = threadIdx.x, lane = tid % kWave, wave = uniform(tid / kWave);
  const int n = uniform(max(0, (int)min((int64_t)used[b], capacity)));
  const int left = min(n, keep);
  if (h == 0 && layer == 0 && tid == 0) used_out[b] = left;
  // The first `free` positions are chosen from, `want` of them.
  const int free = n > keep ? n - min(recent, keep) : 0, want = left - (n - free);
  if constexpr (kHeld) {
    // four at a time: a row has a multiple of 16
    for (int j = 4 * tid; j < n; j += 4 * kThreads)
      *reinterpret_cast<f32x4 *>(sm_w + j) = *reinterpret_cast<const f32x4 *>(w + j);
  }
  // Four weights at a time: a wave alone on its SIMD waits for every read of LDS (one at a
  // time, 16 steps of some 360 cycles where four take as many).
  auto weights4 = [&](int j) { return *reinterpret_cast<const f32x4 *>((kHeld ? sm_w : w) + j); };
  // The wave's stretch of the row, a multiple of 256 positions from the row's start.
  const int stretch = ((n + 4 * kThreads - 1) / (4 * kThreads)) * 4 * kWave;
  const int begin = min(n, wave * stretch), end = min(n, begin + stretch);
  const int last4 = max(n - 1, 0) & ~3;
  const uint64_t lower = ((uint64_t)1 << lane) - 1;
  // For every four positions of the stretch that a lane has: f(j, which of them hold,
  // how many hold before j in this step, how many in all of it).
  auto stretched = [&](auto holds, auto f) {
    for (int j0 = begin; j0 < end; j0 += 4 * kWave) {
      const int j = j0 + 4 * lane;
      const f32x4 x = weights4(min(j, last4));
      bool yes[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) yes[e] = (j + e < end) & holds(j + e, x[e]);
      int before = 0, all = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint64_t mask = __ballot(yes[e]);
        before += __popcll(mask & lower);
        all += __popcll(mask);
      }
      f(j, yes, x, before, all);
    }
  };
  // Exclusive sum over the waves of a number that each has.
  auto waves_before = [&](int v) {
    if (lane == 0) sm_wave[wave] = v;
    __syncthreads();
    int before = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) before += i < wave ? sm_wave[i] : 0;
    return uniform(before);
  };
  // The last of the `want` in this order; what comes before it stays.
  uint64_t least = ~(uint64_t)0;
  if (free > 0 && want > 0) {
    uint32_t prefix = 0, mask = 0;  // leading bits of its key, as far as they are known
    int need = want;                // its rank among the keys that share them
    bool found = false;
    for (int pass = 0; pass < 3 && !found; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
      for (int i = tid; i < kBins; i += kThreads) bins[i] = 0;
      if (tid == 0) sm_candidates = 0;
      __syncthreads();
      for (int j = 4 * tid; j < free; j += 4 * kThreads) {
        const f32x4 x = weights4(j);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t key = key_of(x[e]);
          if ((j + e < free) & ((key & mask) == prefix)) atomicAdd(&bins[(key >> shift) & ((1 << bits) - 1)], 1);
        }
      }
      __syncthreads();
      // From the top: the bin in which the need-th key lies. A thread kOwn bins in a
      // row, the last thread the lowest (with 10 bits the upper half is empty).
      const int *ones = bins + (kBins - kOwn - kOwn * tid);
      int own[kOwn], sum = 0;
#pragma unroll
      for (int i = 0; i < kOwn; ++i) sum += own[i] = ones[kOwn - 1 - i];
      int total;
      int above = wave_prefix(sum, lane, total);
      above += waves_before(total);
      if (above < need && need <= above + sum) {
        int at = 0, count = own[0];
#pragma unroll
        for (int i = 0; i < kOwn - 1; ++i) {
          const bool past = need > above + own[i] && at == i;
          above += past ? own[i] : 0;
          at += past;
          count = past ? own[i + 1] : count;
        }
        sm_found[0] = kBins - 1 - kOwn * tid - at;
        sm_found[1] = need - above;
        sm_found[2] = count;
      }
      __syncthreads();
      prefix |= (uint32_t)uniform(sm_found[0]) << shift;
      mask |= (uint32_t)((1 << bits) - 1) << shift;
      need = uniform(sm_found[1]);
      const int count = uniform(sm_found[2]);
      if (count <= kCandidates) {
        // Few enough: they are gathered, in any order, and each ranked against all.
        for (int j = 4 * tid; j < free; j += 4 * kThreads) {
          const f32x4 x = weights4(j);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t key = key_of(x[e]);
            if ((j + e < free) & ((key & mask) == prefix)) sm_candidate[atomicAdd(&sm_candidates, 1)] = order_of(key, j + e);
          }
        }
        if (tid < kCandidates && tid >= count) sm_candidate[tid] = 0;
        __syncthreads();
        if (tid < count) {
          const uint64_t mine = sm_candidate[tid];
          int rank = 0;
#pragma unroll
          for (int i = 0; i < kCandidates; ++i) rank += sm_candidate[i] > mine;
          if (rank == need - 1) sm_least = mine;
        }
        found = true;
      }
      __syncthreads();
    }
    if (!found) {
      // Many of one weight: the need-th of them in the order of the positions.
      auto equal = [&](int j, float x) { return (j < free) & (key_of(x) == prefix); };
      int mine = 0;
      stretched(equal, [&](int, const bool *, const f32x4 &, int, int all) { mine += all; });
      int seen = waves_before(mine);
      stretched(equal, [&](int j, const bool *yes, const f32x4 &, int before, int all) {
        int rank = seen + before;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (yes[e] && rank == need - 1) sm_least = order_of(prefix, j + e);
          rank += yes[e];
        }
        seen += all;
      });
      __syncthreads();
    }
    least = sm_least;
  } else {
    __syncthreads();  // the weights are in LDS
  }
  // What stays, by the last one's weight t and position: heavier (a NaN is, whose
  // comparison fails) or as heavy and no later.
  const uint32_t least_key = uniform((int)(least >> 32));
  const int least_at = want > 0 ? uniform((int)~(uint32_t)least) : -1;
  const float t = want > 0 ? __uint_as_float(least_key ^ ((int32_t)least_key < 0 ? 0x80000000u : 0xffffffffu)) : INFINITY;
  const bool nans = least_key == 0xffffffffu;
  auto stays = [&](int j, float x) {
    const bool before = j <= least_at, same = nans ? x != x : x == t, above = !nans & !(x <= t);
    return (j >= free) | above | (same & before);
  };
  int mine = 0;
  stretched(stays, [&](int, const bool *, const f32x4 &, int, int all) { mine += all; });
  int done = waves_before(mine);
  stretched(stays, [&](int j, const bool *yes, const f32x4 &x, int before, int all) {
    int at = done + before;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (yes[e]) {
        const uint32_t byte = 4 * (uint32_t)at;
        *reinterpret_cast<int32_t *>(reinterpret_cast<char *>(to) + byte) = j + e;
        *reinterpret_cast<float *>(reinterpret_cast<char *>(w_out) + byte) = x[e];
      }
      at += yes[e];
    }
    done += all;
  });
  for (int j = left + tid; j < keep; j += kThreads) to[j] = -1;
  // zeros behind, four at a time from the next multiple of four
  const int whole = (left + 3) / 4 * 4;
  if (left + tid < whole) w_out[left + tid] = 0.f;
  for (int64_t j = whole + 4 * tid; j < capacity; j += 4 * kThreads)
    *reinterpret_cast<f32x4 *>(w_out + j) = f32x4{0.f, 0.f, 0.f, 0.f};
}

// A thread 16 bytes of K and of V.
constexpr int kMoveThreads = 256;
__global__ void __launch_bounds__(kMoveThreads)
evict_move_kernel(PagedKV kv, int64_t layer_elems, const int32_t *__restrict__ source,
                  const int32_t *__restrict__ target, int target_width, const int32_t *__restrict__ kept, int keep,
                  int dim, int batch) {
  const int units = dim / 8;
  const int to = blockIdx.x * (kMoveThreads / units) + threadIdx.x / units, c = threadIdx.x % units * 8;
  if (to >= keep) return;
  const int h = blockIdx.y;
  const int layer = blockIdx.z / batch, b = blockIdx.z % batch;
  const int from = kept[(((int64_t)layer * batch + b) * kv.heads + h) * keep + to];
  if (from < 0 || (from >> kv.shift) >= kv.width || (to >> kv.shift) >= target_width) return;
  const int64_t old_page = source[(int64_t)b * kv.width + (from >> kv.shift)];
  const int64_t new_page = target[(int64_t)b * target_width + (to >> kv.shift)];
  if (new_page < 0 || new_page >= kv.pages) return;
  const int in_page = (1 << kv.shift) - 1;
  const int64_t at = layer * layer_elems + c;
  const int64_t src = at + (((old_page * kv.heads + h) << kv.shift) + (from & in_page)) * dim;
  const int64_t dst = at + (((new_page * kv.heads + h) << kv.shift) + (to & in_page)) * dim;
  // A position that had no page gives zeros, as it reads: its new page was another's before.
  u32x4 wk{0, 0, 0, 0}, wv{0, 0, 0, 0};
  if (old_page >= 0 && old_page < kv.pages) {
    wk = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(kv.k + src));
    wv = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(kv.v + src));
  }
  *reinterpret_cast<u32x4 *>(kv.k + dst) = wk;
  *reinterpret_cast<u32x4 *>(kv.v + dst) = wv;
}

}  // namespace
}  // namespace lm

using namespace lm;

extern "C" int lm_kv_evict(const lm_kv_evict_args *args, void *stream) {
  LM_REQUIRE(args);
  const auto &[k_pages, v_pages, source, target, width, target_width, pages, page, used, weights, layers, batch, heads,
               head_dim, keep, recent, weights_out, kept, used_out] = *args;
  LM_REQUIRE(layers > 0 && batch >= 0 && heads > 0 && heads <= 65535 && batch <= 65535 && layers <= 65535 &&
             layers * batch <= 65535 && keep > 0 && recent >= 0 && recent <= keep && target_width > 0);
  const int status = paged_args_ok(width, pages, page, head_dim);
  if (status != LM_OK) return status;
  LM_REQUIRE(keep <= width * page && target_width <= ((int64_t)1 << 30) / page);
  if (batch == 0) return LM_OK;
  LM_REQUIRE(k_pages && v_pages && source && target && used && weights && weights_out && kept && used_out);
  LM_REQUIRE(aligned16(k_pages) && aligned16(v_pages) && aligned16(weights) && aligned16(weights_out));
  hipStream_t s = (hipStream_t)stream;
  const int64_t capacity = width * page;
  const bool held = capacity <= kHeldWeights;
  LM_REQUIRE(held || weights != weights_out);
  LM_REQUIRE(in_place_or_apart(weights, weights_out, layers * batch * heads * capacity * 4));
  // One step of four weights a thread, or two: a wave alone on its SIMD waits for every
  // instruction. One row of 4096 weights 12.4 us with 256 threads, 9.2 with 512; 1024 such
  // rows 20.5 and 22.0 (bytes in and out 7, the rest latency).
  const auto select = !held              ? evict_select_kernel<1024, false>
                      : capacity <= 1024 ? evict_select_kernel<256, true>
                      : capacity <= 4096 ? evict_select_kernel<512, true>
                                         : evict_select_kernel<1024, true>;
  select<<<dim3((unsigned)heads, (unsigned)batch, (unsigned)layers),
           capacity <= 1024 ? 256 : capacity <= 4096 ? 512 : 1024, held ? capacity * 4 : 0, s>>>(
      used, weights, capacity, (int)keep, (int)recent, weights_out, kept, used_out);
  LM_CHECK_LAUNCH();
  const PagedKV kv{(bf16 *)k_pages, (bf16 *)v_pages, pages, (int)width, page_shift(page), (int)heads};
  const int64_t per_block = kMoveThreads / (head_dim / 8);
  evict_move_kernel<<<dim3((unsigned)cdiv(keep, per_block), (unsigned)heads, (unsigned)(layers * batch)),
                      kMoveThreads, 0, s>>>(kv, pages * heads * page * head_dim, source, target, (int)target_width,
                                            kept, (int)keep, (int)head_dim, (int)batch);
  LM_CHECK_LAUNCH();
  return LM_OK;
}
