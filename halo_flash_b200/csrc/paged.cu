// A paged K/V cache: the plan of a step (block tables and slot maps from lengths) and the store of its new rows.
//
// Pages hold 2^page_shift tokens. Request r has past[r] tokens in the first ceil(past[r] / page) pages of its table
// row and gets fresh[r] more; it needs ceil((past + fresh) / page) - ceil(past / page) new pages, which come from the
// list of free pages in the order of the requests.
#include "common.cuh"
#include "kernels.h"

namespace halo_b200 {

namespace {

// ---- plan -------------------------------------------------------------------------------------------------
// Latency bound: a serving step has at most a few thousand requests and tokens, tens of kilobytes in all. One
// launch, no atomics and no second pass: every CTA reads all lengths and builds the two prefix sums (tokens, new
// pages) in its own shared memory, then takes its share of the tokens and of the new pages, each of which finds
// its request by bisection. A token of a new page takes the page from the free list itself, not from the table that
// some other CTA is writing. 8 requests 2.5 us, 1024 requests with 65536 tokens 4.4 us.
constexpr unsigned kPlanThreads = 512;

// The first index whose entry is greater than x, less one (a[0] == 0 <= x).
__device__ __forceinline__ uint32_t find(const uint32_t* a, uint32_t n, uint32_t x) {
  uint32_t lo = 0, hi = n;  // a[lo] <= x < a[hi]
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) >> 1;
    if (a[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(const PlanArgs p) {
  extern __shared__ uint32_t plan_smem[];
  uint32_t* cu = plan_smem;                 // [batch + 1]
  uint32_t* first = plan_smem + p.batch + 1;  // [batch + 1]
  __shared__ unsigned long long warp_tok[kPlanThreads / 32], warp_page[kPlanThreads / 32];
  __shared__ uint32_t refused;
  pdl_begin();
  const uint32_t page = 1u << p.page_shift, tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
  const uint32_t per = (p.batch + kPlanThreads - 1) / kPlanThreads;
  const uint32_t r0 = min(p.batch, tid * per), r1 = min(p.batch, r0 + per);
  if (tid == 0) refused = 0;

  auto pages_of = [&](uint32_t past, uint32_t fresh, uint32_t* held) -> uint32_t {
    // lengths count in 64 bits: past + fresh may pass 32
    *held = static_cast<uint32_t>((static_cast<unsigned long long>(past) + page - 1) >> p.page_shift);
    const unsigned long long want = (static_cast<unsigned long long>(past) + fresh + page - 1) >> p.page_shift;
    if (want > p.table_cols) return 0xFFFFFFFFu;  // does not fit its table row
    return static_cast<uint32_t>(want) - *held;
  };

  unsigned long long toks = 0, news = 0;
  for (uint32_t r = r0; r < r1; ++r) {
    uint32_t held;
    const uint32_t fresh = p.fresh[r], need = pages_of(p.past[r], fresh, &held);
    toks += fresh;
    if (need != 0xFFFFFFFFu) news += need;
  }
  unsigned long long it = toks, ip = news;  // inclusive sums over the warp
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long t = __shfl_up_sync(kFullMask, it, o), q = __shfl_up_sync(kFullMask, ip, o);
    if (lane >= static_cast<unsigned>(o)) it += t, ip += q;
  }
  if (lane == 31) warp_tok[warp] = it, warp_page[warp] = ip;
  __syncthreads();
  unsigned long long bt = it - toks, bp = ip - news;
  for (uint32_t w = 0; w < warp; ++w) bt += warp_tok[w], bp += warp_page[w];
  const unsigned long long cap = 0xFFFFFFFFull;
  for (uint32_t r = r0; r < r1; ++r) {
    uint32_t held;
    const uint32_t fresh = p.fresh[r], past = p.past[r], need = pages_of(past, fresh, &held);
    cu[r] = static_cast<uint32_t>(min(bt, cap));
    first[r] = static_cast<uint32_t>(min(bp, cap));
    const bool fits = need != 0xFFFFFFFFu && (need == 0 || bp + need <= p.n_free);
    if (blockIdx.x == 0) {
      if (p.cu) p.cu[r] = cu[r];
      if (p.kv_len) p.kv_len[r] = fits ? past + fresh : past;
      if (!fits) atomicAdd(&refused, 1u);  // a count: its order does not matter
    }
    bt += fresh;
    if (need != 0xFFFFFFFFu) bp += need;
  }
  if (r1 == p.batch && r0 < r1) cu[p.batch] = static_cast<uint32_t>(min(bt, cap)), first[p.batch] = static_cast<uint32_t>(min(bp, cap));
  if (p.batch == 0 && tid == 0) cu[0] = first[0] = 0;
  __syncthreads();
  const uint32_t total = cu[p.batch], pages = min(first[p.batch], p.n_free);

  // Whether request r gets its pages. What is taken is a prefix of the free list: once one request does not fit,
  // none behind it that needs a page does.
  const uint32_t step = gridDim.x * kPlanThreads, g = blockIdx.x * kPlanThreads + tid;
  for (uint32_t i = g; i < pages; i += step) {
    const uint32_t r = find(first, p.batch, i);
    if (first[r + 1] > p.n_free) continue;
    uint32_t held;
    pages_of(p.past[r], p.fresh[r], &held);
    p.table[r * p.table_stride + held + (i - first[r])] = p.free_pages[i];
  }
  for (uint32_t t = g; t < p.tokens; t += step) {
    int64_t slot = -1;
    uint32_t pos = 0;
    if (t < total) {
      const uint32_t r = find(cu, p.batch, t);
      uint32_t held;
      const uint32_t past = p.past[r], need = pages_of(past, p.fresh[r], &held);
      pos = past + (t - cu[r]);
      if (need != 0xFFFFFFFFu && (need == 0 || first[r + 1] <= p.n_free)) {
        const uint32_t col = pos >> p.page_shift;
        const int32_t block = col < held ? p.table[r * p.table_stride + col] : p.free_pages[first[r] + (col - held)];
        slot = static_cast<int64_t>(block) * page + (pos & (page - 1));
      }
    }
    p.slot[t] = slot;
    if (p.pos) p.pos[t] = pos;
  }
  if (blockIdx.x == 0 && tid == 0) {
    if (p.cu) p.cu[p.batch] = total;
    if (p.status) {
      // pages taken: what the last request that got its pages ends at
      uint32_t taken = first[p.batch];
      if (taken > p.n_free) {
        uint32_t lo = 0, hi = p.batch;  // first[lo] <= n_free < first[hi]
        while (hi - lo > 1) {
          const uint32_t mid = (lo + hi) >> 1;
          if (first[mid] <= p.n_free) lo = mid;
          else hi = mid;
        }
        taken = first[lo];
      }
      p.status[0] = taken;
      p.status[1] = refused;
      p.status[2] = total;
    }
  }
}

// ---- store ------------------------------------------------------------------------------------------------
// HBM bound: each row is read once and written once. A thread moves one octet (8 values) of K and the same octet of
// V, both loads in flight before either store; neighbouring threads take neighbouring octets of a row. 65536 rows of
// 2 x 256: 42.9 us from 16-bit to 16-bit types (6.3 TB/s), 62.0 from fp32 to bf16 (6.5), 86.8 from fp32 to fp32 (6.2).
template <typename IT, typename OT, bool VEC>
__global__ void __launch_bounds__(kBlock) paged_store_kernel(const StoreArgs a) {
  pdl_begin();
  constexpr uint32_t kW = VEC ? 8 : 1;
  const uint32_t per_head = a.dim / kW, per_row = a.heads * per_head;
  const uint64_t total = static_cast<uint64_t>(a.tokens) * per_row;
  const uint64_t limit = static_cast<uint64_t>(a.pages) << a.page_shift;
  for (uint64_t i = blockIdx.x * static_cast<uint64_t>(kBlock) + threadIdx.x; i < total; i += static_cast<uint64_t>(gridDim.x) * kBlock) {
    const uint32_t t = static_cast<uint32_t>(i / per_row), c = static_cast<uint32_t>(i - static_cast<uint64_t>(t) * per_row);
    const uint32_t h = c / per_head, e = (c - h * per_head) * kW;
    const int64_t slot = a.slot[t];
    if (slot < 0 || static_cast<uint64_t>(slot) >= limit) continue;
    const uint64_t to = (static_cast<uint64_t>(slot) >> a.page_shift) * a.page_stride +
                        (static_cast<uint64_t>(slot) & ((1u << a.page_shift) - 1)) * a.row_stride + h * a.head_stride + e;
    const IT* k = static_cast<const IT*>(a.src[0]) + t * a.src_row[0] + h * a.src_head[0] + e;
    const IT* v = static_cast<const IT*>(a.src[1]) + t * a.src_row[1] + h * a.src_head[1] + e;
    OT* ko = static_cast<OT*>(a.dst[0]) + to;
    OT* vo = static_cast<OT*>(a.dst[1]) + to;
    if constexpr (VEC) {
      const Raw<IT> rk = raw_load(k), rv = raw_load(v);
      oct_store(ko, raw_unpack(rk));
      oct_store(vo, raw_unpack(rv));
    } else {
      *ko = from_f32<OT>(to_f32(*k));
      *vo = from_f32<OT>(to_f32(*v));
    }
  }
}

template <typename IT, typename OT>
cudaError_t LaunchStore(const StoreArgs& a, cudaStream_t s) {
  const uint64_t n = static_cast<uint64_t>(a.tokens) * a.heads * (a.vec ? a.dim / 8 : a.dim);
  uint64_t grid = (n + kBlock - 1) / kBlock;
  if (grid > 148u * 64u) grid = 148u * 64u;
  if (a.vec) return LaunchKernel(paged_store_kernel<IT, OT, true>, static_cast<unsigned>(grid), kBlock, 0, s, a);
  return LaunchKernel(paged_store_kernel<IT, OT, false>, static_cast<unsigned>(grid), kBlock, 0, s, a);
}

}  // namespace

cudaError_t LaunchPagedPlan(const PlanArgs& a, cudaStream_t s) {
  const unsigned smem = 8u * (a.batch + 1);
  if (smem > 48u * 1024u) {
    // for the largest batch, always: calls from several threads set the same limit, none one that is too low for another's launch
    const cudaError_t e = cudaFuncSetAttribute(paged_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(8u * (kMaxPlanBatch + 1)));
    if (e != cudaSuccess) return e;
  }
  // new pages <= tokens + batch, but `tokens` may be shorter than the lengths say; the loops stride, so any grid is right
  uint64_t grid = (static_cast<uint64_t>(a.tokens) + kPlanThreads - 1) / kPlanThreads;
  if (grid < 1) grid = 1;
  if (grid > 148) grid = 148;
  return LaunchKernel(paged_plan_kernel, static_cast<unsigned>(grid), kPlanThreads, smem, s, a);
}

cudaError_t LaunchPagedStore(const StoreArgs& a, cudaStream_t s) {
  switch (a.src_dtype * 3 + a.dst_dtype) {
    case kF32 * 3 + kF32: return LaunchStore<float, float>(a, s);
    case kF32 * 3 + kF16: return LaunchStore<float, f16>(a, s);
    case kF32 * 3 + kBF16: return LaunchStore<float, bf16>(a, s);
    case kF16 * 3 + kF16: return LaunchStore<f16, f16>(a, s);
    case kF16 * 3 + kBF16: return LaunchStore<f16, bf16>(a, s);
    case kBF16 * 3 + kF16: return LaunchStore<bf16, f16>(a, s);
    case kBF16 * 3 + kBF16: return LaunchStore<bf16, bf16>(a, s);
  }
  return cudaErrorInvalidValue;
}

}  // namespace halo_b200
