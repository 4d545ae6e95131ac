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

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / kWave;
constexpr int kBins = 2048;

// Larger floats, larger keys: -0 as 0, a NaN above every number.
__device__ __forceinline__ uint32_t key_of(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.f);
  return u ^ ((int32_t)u < 0 ? 0xffffffffu : 0x80000000u);
}

// Exclusive prefix over the workgroup of each thread's count, and the total.
__device__ __forceinline__ int block_prefix(int v, int *sm, int &total) {
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  int x = v;
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const int y = __shfl_up(x, d, kWave);
    if (lane >= d) x += y;
  }
  __syncthreads();
  if (lane == kWave - 1) sm[wave] = x;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const int c = sm[w];
    before += w < wave ? c : 0;
    total += c;
  }
  return before + x - v;
}

__global__ void __launch_bounds__(kThreads)
evict_select_kernel(const int32_t *__restrict__ used, const float *weights, int64_t capacity, int keep, int recent,
                    float *weights_out, int32_t *__restrict__ kept, int32_t *__restrict__ used_out) {
  __shared__ int bins[kBins];
  __shared__ int sm[kWaves];
  __shared__ int sm_found[2];
  const int h = blockIdx.x, heads = gridDim.x;
  const int64_t b = blockIdx.y, batch = gridDim.y, layer = blockIdx.z;
  const int64_t row = (layer * batch + b) * heads + h;
  const float *w = weights + row * capacity;
  float *w_out = weights_out + row * capacity;
  int32_t *to = kept + row * keep;
  const int n = max(0, (int)min((int64_t)used[b], capacity));
  const int left = min(n, keep);
  if (h == 0 && layer == 0 && threadIdx.x == 0) used_out[b] = left;
  // The first `free` positions are chosen from, `want` of them.
  const int free = n > keep ? n - min(recent, keep) : 0, want = left - (n - free);
  uint32_t prefix = 0, mask = 0;
  int need = want;  // of the keys that share the prefix found so far
  if (free > 0 && want > 0) {
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, count = pass == 2 ? 1 << 10 : 1 << 11;
      for (int i = threadIdx.x; i < count; i += kThreads) bins[i] = 0;
      __syncthreads();
      for (int j = threadIdx.x; j < free; j += kThreads) {
        const uint32_t key = key_of(w[j]);
        if ((key & mask) == prefix) atomicAdd(&bins[(key >> shift) & (count - 1)], 1);
      }
      __syncthreads();
      // From the top: the bin in which the need-th key lies. A thread two bins.
      const int hi = count - 1 - 2 * (int)threadIdx.x;
      const int c1 = hi >= 0 ? bins[hi] : 0, c2 = hi >= 1 ? bins[hi - 1] : 0;
      int total;
      const int above = block_prefix(c1 + c2, sm, total);
      if (above < need && need <= above + c1 + c2) {
        const bool first = need <= above + c1;
        sm_found[0] = first ? hi : hi - 1;
        sm_found[1] = need - above - (first ? 0 : c1);
      }
      __syncthreads();
      prefix |= (uint32_t)sm_found[0] << shift;
      mask |= (uint32_t)(count - 1) << shift;
      need = sm_found[1];
      __syncthreads();
    }
  }
  // In order: the kept indices and their weights. A chunk is read before it is
  // written, and what is kept never moves up, so the weights may be their own output.
  int done = 0, ties = 0;  // kept and taken from the equal ones so far
  for (int j0 = 0; j0 < n; j0 += kThreads) {
    const int j = j0 + threadIdx.x;
    const float x = j < n ? w[j] : 0.f;
    const uint32_t key = key_of(x);
    const bool equal = j < free && want > 0 && key == prefix;
    int equals = 0, total = 0;
    const int rank = ties + block_prefix(equal ? 1 : 0, sm, equals);
    const bool stays = j < n && (j >= free || (want > 0 && key > prefix) || (equal && rank < need));
    const int at = done + block_prefix(stays ? 1 : 0, sm, total);
    ties += equals;
    done += total;
    if (stays) {
      to[at] = j;
      w_out[at] = x;
    }
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

extern "C" int lm_kv_evict(void *k_pages, void *v_pages, const int32_t *source, const int32_t *target, int64_t width,
                           int64_t target_width, int64_t pages, int64_t page, const int32_t *used,
                           const float *weights, int64_t layers, int64_t batch, int64_t heads, int64_t head_dim,
                           int64_t keep, int64_t recent, float *weights_out, int32_t *kept, int32_t *used_out,
                           void *stream) {
  LM_REQUIRE(layers > 0 && batch >= 0 && heads > 0 && heads <= 65535 && batch <= 65535 && layers <= 65535 &&
             layers * batch <= 65535 && keep > 0 && recent >= 0 && recent <= keep && target_width > 0);
  const int status = paged_args_ok(width, pages, page, head_dim);
  if (status != LM_OK) return status;
  LM_REQUIRE(keep <= width * page && target_width <= ((int64_t)1 << 30) / page);
  if (batch == 0) return LM_OK;
  LM_REQUIRE(k_pages && v_pages && source && target && used && weights && weights_out && kept && used_out);
  LM_REQUIRE(aligned16(k_pages) && aligned16(v_pages));
  hipStream_t s = (hipStream_t)stream;
  evict_select_kernel<<<dim3((unsigned)heads, (unsigned)batch, (unsigned)layers), kThreads, 0, s>>>(
      used, weights, width * page, (int)keep, (int)recent, weights_out, kept, used_out);
  LM_CHECK_LAUNCH();
  const PagedKV kv{(bf16 *)k_pages, (bf16 *)v_pages, pages, (int)width, page_shift(page), (int)heads};
  const int64_t per_block = kMoveThreads / (head_dim / 8);
  evict_move_kernel<<<dim3((unsigned)cdiv(keep, per_block), (unsigned)heads, (unsigned)(layers * batch)),
                      kMoveThreads, 0, s>>>(kv, pages * heads * page * head_dim, source, target, (int)target_width,
                                            kept, (int)keep, (int)head_dim, (int)batch);
  LM_CHECK_LAUNCH();
  return LM_OK;
}
