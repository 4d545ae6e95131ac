// Eviction from a paged cache by weight: of a row's n = used[b] positions, per
// layer and KV head, the `recent` last ones and the heaviest of the others stay,
// `keep` in all, in their order.
//
// Selection, one workgroup per (layer, row, KV head): the keep-th heaviest weight
// by radix over the weights as ordered integers (11, 11 and 10 bits from the top,
// counts in LDS), then one pass in order that writes the kept indices and weights:
// those above the threshold, and of those equal to it the first. Whole numbers
// throughout, so the order of the counting does not show.
//
// Move: every kept position's K and V go from the row's pages to their place in the
// target's pages, a second launch over (kept, KV head, layer and row). Out of place,
// so that pages which another row shares are left as they are and no order of the
// moves matters.
//
// The reference holds every position to the end (litemoe/cache.py:7-20).
#include "paged.h"

namespace lm {
namespace {

constexpr int kBits = 11, kBins = 1 << kBits;

// Larger floats, larger keys: -0 as 0, a NaN above every number.
__device__ __forceinline__ uint32_t key_of(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.f);
  return u ^ ((int32_t)u < 0 ? 0xffffffffu : 0x80000000u);
}

// Sum of the lanes below this one, by shuffles over the wave.
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

// kThreads threads take kPer weights each at a time, thread t those at t, t + kThreads,
// ... of the chunk. A row of one chunk is read once and stays in registers.
template <int kThreads, int kPer>
__global__ void __launch_bounds__(kThreads)
evict_select_kernel(const int32_t *__restrict__ used, const float *weights, int64_t capacity, int keep, int recent,
                    float *weights_out, int32_t *__restrict__ kept, int32_t *__restrict__ used_out) {
  constexpr int kWaves = kThreads / kWave, kChunk = kThreads * kPer, kOwn = kBins / kThreads;
  static_assert(kWaves * kPer <= 4 * kWave, "a wave scans the chunk's counts, four a lane");
  __shared__ __attribute__((aligned(16))) int bins[kBins];
  __shared__ int sm_wave[kWaves];
  __shared__ int sm_found[2];
  __shared__ int sm_count[2][kPer * kWaves];  // by (round, wave): equal ones, then kept ones
  __shared__ int sm_total[2];
  const int h = blockIdx.x, heads = gridDim.x;
  const int64_t b = blockIdx.y, batch = gridDim.y, layer = blockIdx.z;
  const int64_t row = (layer * batch + b) * heads + h;
  const float *w = weights + row * capacity;
  float *w_out = weights_out + row * capacity;
  int32_t *to = kept + row * keep;
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int n = max(0, (int)min((int64_t)used[b], capacity));
  const int left = min(n, keep);
  if (h == 0 && layer == 0 && threadIdx.x == 0) used_out[b] = left;
  // The first `free` positions are chosen from, `want` of them.
  const int free = n > keep ? n - min(recent, keep) : 0, want = left - (n - free);
  const bool choose = free > 0 && want > 0;
  float x[kPer];
  auto load = [&](int j0) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int j = j0 + i * kThreads + threadIdx.x;
      x[i] = j < n ? w[j] : 0.f;
    }
  };
  load(0);
  // The threshold: bits of the want-th largest key from the top, and how many of
  // its equals are wanted.
  uint32_t prefix = 0, mask = 0;
  int need = want;
  if (choose) {
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
#pragma unroll
      for (int i = 0; i < kBins; i += kThreads) bins[i + threadIdx.x] = 0;
      __syncthreads();
      for (int j0 = 0; j0 < free; j0 += kChunk) {
        if (n > kChunk) load(j0);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const int j = j0 + i * kThreads + threadIdx.x;
          const uint32_t key = key_of(x[i]);
          if (j < free && (key & mask) == prefix) atomicAdd(&bins[(key >> shift) & ((1 << bits) - 1)], 1);
        }
      }
      __syncthreads();
      // From the top: the bin in which the need-th key lies. A thread kOwn bins in a
      // row, the last thread the lowest (with 10 bits the upper half is empty).
      const int top = kBins - 1 - kOwn * (int)threadIdx.x;
      int own[kOwn], sum = 0;
#pragma unroll
      for (int i = 0; i < kOwn; ++i) sum += own[i] = bins[top - i];
      int total;
      int above = wave_prefix(sum, lane, total);
      if (lane == 0) sm_wave[wave] = total;
      __syncthreads();
#pragma unroll
      for (int v = 0; v < kWaves; ++v) above += v < wave ? sm_wave[v] : 0;
      if (above < need && need <= above + sum) {
        int at = 0;
#pragma unroll
        for (int i = 0; i < kOwn - 1; ++i) {
          const bool past = need > above + own[i] && at == i;
          above += past ? own[i] : 0;
          at += past;
        }
        sm_found[0] = top - at;
        sm_found[1] = need - above;
      }
      __syncthreads();
      prefix |= (uint32_t)sm_found[0] << shift;
      mask |= (uint32_t)((1 << bits) - 1) << shift;
      need = sm_found[1];
    }
  }
  // In order: the kept indices and their weights. A chunk is read before it is
  // written, and what is kept never moves up, so the weights may be their own output.
  const uint64_t below = ((uint64_t)1 << lane) - 1;
  // Exclusive sums of a chunk's counts in the order of the positions, by the first wave.
  auto scan = [&](int *count, int *chunk_total) {
    __syncthreads();
    if (wave == 0) {
      int c[4], sum = 0, total;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = 4 * lane + i;
        c[i] = at < kPer * kWaves ? count[at] : 0;
        sum += c[i];
      }
      int before = wave_prefix(sum, lane, total);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = 4 * lane + i;
        if (at < kPer * kWaves) count[at] = before;
        before += c[i];
      }
      if (lane == 0) *chunk_total = total;
    }
    __syncthreads();
  };
  int done = 0, ties = 0;  // kept, and equal ones seen, in the chunks before
  for (int j0 = 0; j0 < n; j0 += kChunk) {
    if (n > kChunk) load(j0);
    uint64_t equal[kPer], stay[kPer];
    if (choose) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int j = j0 + i * kThreads + threadIdx.x;
        equal[i] = __ballot(j < free && key_of(x[i]) == prefix);
        if (lane == 0) sm_count[0][i * kWaves + wave] = __popcll(equal[i]);
      }
      scan(sm_count[0], &sm_total[0]);
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int j = j0 + i * kThreads + threadIdx.x;
      bool stays = j < n;
      if (choose && j < free) {
        const bool same = (equal[i] >> lane) & 1;
        const int rank = ties + sm_count[0][i * kWaves + wave] + __popcll(equal[i] & below);
        stays = same ? rank < need : key_of(x[i]) > prefix;
      } else if (j < free) {
        stays = false;
      }
      stay[i] = __ballot(stays);
      if (lane == 0) sm_count[1][i * kWaves + wave] = __popcll(stay[i]);
    }
    scan(sm_count[1], &sm_total[1]);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if ((stay[i] >> lane) & 1) {
        const int at = done + sm_count[1][i * kWaves + wave] + __popcll(stay[i] & below);
        to[at] = j0 + i * kThreads + threadIdx.x;
        w_out[at] = x[i];
      }
    }
    if (choose) ties += sm_total[0];
    done += sm_total[1];
    __syncthreads();
  }
  for (int j = left + threadIdx.x; j < keep; j += kThreads) to[j] = -1;
  __syncthreads();
  for (int64_t j = left + threadIdx.x; j < capacity; j += kThreads) w_out[j] = 0.f;
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
  if (old_page < 0 || old_page >= kv.pages || new_page < 0 || new_page >= kv.pages) return;
  const int in_page = (1 << kv.shift) - 1;
  const int64_t at = layer * layer_elems + c;
  const int64_t src = at + (((old_page * kv.heads + h) << kv.shift) + (from & in_page)) * dim;
  const int64_t dst = at + (((new_page * kv.heads + h) << kv.shift) + (to & in_page)) * dim;
  const u32x4 wk = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(kv.k + src));
  const u32x4 wv = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(kv.v + src));
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
  LM_REQUIRE(aligned16(k_pages) && aligned16(v_pages));
  hipStream_t s = (hipStream_t)stream;
  const int64_t capacity = width * page;
  auto select = capacity <= 1024 ? evict_select_kernel<256, 4>
                : capacity <= 4096 ? evict_select_kernel<256, 16>
                                   : evict_select_kernel<1024, 8>;
  select<<<dim3((unsigned)heads, (unsigned)batch, (unsigned)layers), capacity <= 4096 ? 256 : 1024, 0, s>>>(
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
