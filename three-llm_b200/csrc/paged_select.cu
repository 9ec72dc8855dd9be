// Choosing the pages that a sparse decode step reads. A page's score bounds
// the summed dot products of a kv head's query heads with any of its keys:
//
//   s = sum_h sum_d (q_hd > 0 ? q_hd high_d : q_hd low_d) = sum_d (P_d high_d + N_d low_d),
//   P_d = sum_h max(q_hd, 0), N_d = sum_h min(q_hd, 0)
//
// one dot product of length 2 D per page whatever the group size. It is formed
// in 64 bits: the choice is a whole number that a rounding next to the border
// would change, and after rounding the sum once to 32 bits two ways of adding
// it up agree.
#include <math.h>

#include "paged.cuh"

namespace tla {

namespace {

constexpr int kScoreThreads = 256;
constexpr int kScorePages = 64;  // pages per block
constexpr int kPickThreads = 256;

// Larger scores have larger keys, and every score a key above 0.
__device__ __forceinline__ uint32_t rank_of(float s) {
  const uint32_t u = __float_as_uint(s + 0.f);  // (-0 ranks as +0)
  const uint32_t r = u & 0x80000000u ? ~u : u | 0x80000000u;
  return r == 0u ? 1u : r;
}

struct PageRange {
  int begin, n;  // the pages that hold [window start, pos]
};
__device__ __forceinline__ PageRange page_range(const PagedArgs& p, int pos) {
  int lo, hi;
  if (!paged_range(p, pos, &lo, &hi)) return {0, 0};
  return {lo >> p.page_shift, (hi >> p.page_shift) - (lo >> p.page_shift) + 1};
}

// ranks[b][kvh][i]: page begin + i; the pages that always take part get the
// highest ranks. A warp per page.
template <typename IO, typename CT>
__global__ void __launch_bounds__(kScoreThreads)
    paged_score_kernel(PagedArgs p, const IO* __restrict__ query, int first, int last, int count,
                       uint32_t* __restrict__ ranks) {
  extern __shared__ double vec[];  // [2][D]: N, then P, as the bounds' order
  griddep_wait();
  griddep_launch_dependents();
  const int D = p.a.D, G = p.a.G, Hk = p.a.Hk;
  const int kvh = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int b = blockIdx.z; b < p.batch; b += gridDim.z) {
    const PageRange r = page_range(p, p.positions[b]);
    if (r.n <= count) continue;  // all of them are taken
    const int from = blockIdx.x * kScorePages, to = min(r.n, from + kScorePages);
    if (from >= to) continue;
    __syncthreads();
    for (int d = threadIdx.x; d < D; d += kScoreThreads) {
      double neg = 0, pos = 0;
      for (int g = 0; g < G; ++g) {
        const float q = to_f32(query[(static_cast<int64_t>(b) * p.a.Hq + kvh * G + g) * D + d]);
        neg += fminf(q, 0.f);
        pos += fmaxf(q, 0.f);
      }
      vec[d] = neg;
      vec[D + d] = pos;
    }
    __syncthreads();
    uint32_t* out = ranks + (static_cast<int64_t>(b) * Hk + kvh) * p.width;
    for (int i = from + warp; i < to; i += kScoreThreads / 32) {
      if (i < first || i >= r.n - last) {
        if (lane == 0) out[i] = 0xffffffffu;
        continue;
      }
      const int page = pool_page(p, b, r.begin + i);
      if (page < 0) {
        if (lane == 0) out[i] = 0u;
        continue;
      }
      const CT* at = static_cast<const CT*>(p.bounds) + (static_cast<int64_t>(page) * Hk + kvh) * 2 * D;
      double s = 0;
      for (int d = lane; d < 2 * D; d += 32) s = fma(vec[d], static_cast<double>(to_f32(at[d])), s);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      if (lane == 0) out[i] = min(rank_of(static_cast<float>(s)), 0xfffffffeu);
    }
  }
}

// The `count` highest ranks, ties to the lower page, in page order: a block
// per (sequence, kv head). Four 8-bit passes find the lowest rank that is
// taken and how many pages of exactly that rank are; one more writes the list.
__global__ void __launch_bounds__(kPickThreads)
    paged_pick_kernel(PagedArgs p, const uint32_t* __restrict__ ranks, int count, int32_t* __restrict__ pages_out) {
  __shared__ int bins[256];
  __shared__ int warp_sum_s[2][kPickThreads / 32];
  __shared__ uint32_t prefix_s;
  __shared__ int want_s;
  griddep_wait();
  griddep_launch_dependents();
  const int Hk = p.a.Hk, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int b = blockIdx.x / Hk;
  const int pos = p.positions[b];
  const PageRange r = page_range(p, pos);
  int32_t* out = pages_out + static_cast<int64_t>(blockIdx.x) * count;
  if (r.n == 0 && pos >= 0 && tid == 0) report_error(p.a.error, TLA_ERR_POSITION);
  if (r.n <= count) {
    for (int i = tid; i < count; i += kPickThreads) out[i] = i < r.n ? r.begin + i : -1;
    return;
  }
  const uint32_t* rank = ranks + static_cast<int64_t>(blockIdx.x) * p.width;
  uint32_t prefix = 0;
  int want = count;  // pages still to take among those that share the prefix
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += kPickThreads) bins[i] = 0;
    __syncthreads();
    for (int i = tid; i < r.n; i += kPickThreads) {
      const uint32_t v = rank[i];
      if (shift == 24 || v >> (shift + 8) == prefix) atomicAdd(&bins[(v >> shift) & 255], 1);
    }
    __syncthreads();
    if (tid == 0) {
      int bin = 255;
      while (bin > 0 && bins[bin] < want) want -= bins[bin--];
      prefix_s = prefix << 8 | static_cast<uint32_t>(bin);
      want_s = want;
    }
    __syncthreads();
    prefix = prefix_s;
    want = want_s;
  }
  int taken = 0, equal = 0;  // before this round of pages
  for (int base = 0; base < r.n; base += kPickThreads) {
    const int i = base + tid;
    const uint32_t v = i < r.n ? rank[i] : 0u;
    const bool above = i < r.n && v > prefix, same = i < r.n && v == prefix;
    const unsigned same_mask = __ballot_sync(0xffffffffu, same);
    if (lane == 0) warp_sum_s[0][warp] = __popc(same_mask);
    __syncthreads();
    int eq = equal + __popc(same_mask & ((1u << lane) - 1));
    int eq_all = 0;
    for (int w = 0; w < kPickThreads / 32; ++w) {
      if (w < warp) eq += warp_sum_s[0][w];
      eq_all += warp_sum_s[0][w];
    }
    const bool take = above || (same && eq < want);
    const unsigned take_mask = __ballot_sync(0xffffffffu, take);
    if (lane == 0) warp_sum_s[1][warp] = __popc(take_mask);
    __syncthreads();
    int at = taken + __popc(take_mask & ((1u << lane) - 1));
    int all = 0;
    for (int w = 0; w < kPickThreads / 32; ++w) {
      if (w < warp) at += warp_sum_s[1][w];
      all += warp_sum_s[1][w];
    }
    if (take) out[at] = r.begin + i;
    taken += all;
    equal += eq_all;
    __syncthreads();
  }
}

template <typename IO, typename CT>
cudaError_t select_t(const PagedArgs& p, const void* query, int first, int last, int32_t* pages_out, int count,
                     uint32_t* ranks, cudaStream_t stream) {
  const int most = min(p.width, (p.capacity + (1 << p.page_shift) - 1) >> p.page_shift);
  if (most > count) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((most + kScorePages - 1) / kScorePages, p.a.Hk, min(p.batch, 65535));
    cfg.blockDim = dim3(kScoreThreads);
    cfg.dynamicSmemBytes = 2 * p.a.D * sizeof(double);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, paged_score_kernel<IO, CT>, p, static_cast<const IO*>(query), first,
                                             last, count, ranks);
    if (e != cudaSuccess) return e;
  }
  return launch_pdl(paged_pick_kernel, static_cast<unsigned>(p.batch) * p.a.Hk, kPickThreads, 0, stream, p,
                    static_cast<const uint32_t*>(ranks), count, pages_out);
}

}  // namespace

size_t paged_select_workspace(const tla_paged* P, int batch, int width) {
  return P->pool.bounds ? static_cast<size_t>(batch) * P->base.Hk * width * sizeof(uint32_t) : 0;
}

cudaError_t launch_paged_select(const tla_paged* P, const PagedArgs& p, const void* query, int first, int last,
                                int32_t* pages_out, int count, void* workspace, cudaStream_t stream) {
  uint32_t* ranks = static_cast<uint32_t*>(workspace);
  if (P->io == kFp16) return select_t<__half, __half>(p, query, first, last, pages_out, count, ranks, stream);
  if (P->io == kBf16)
    return select_t<__nv_bfloat16, __nv_bfloat16>(p, query, first, last, pages_out, count, ranks, stream);
  if (P->kept == kFp16) return select_t<float, __half>(p, query, first, last, pages_out, count, ranks, stream);
  if (P->kept == kBf16) return select_t<float, __nv_bfloat16>(p, query, first, last, pages_out, count, ranks, stream);
  return select_t<float, float>(p, query, first, last, pages_out, count, ranks, stream);
}

}  // namespace tla
