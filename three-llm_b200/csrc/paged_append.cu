// Appending rows of [Q | K | V] to a paged cache (the copy-KV and query
// kernels of TSLAttention, packages/three-llm/src/tsl/TSLAttention.ts:252-304,
// with the slot looked up in a page table):
//
//   x <- x / sqrt(mean(x^2) + eps) * w          QK-norm (vNorm: w = 1)
//   (x_j, x_j+h) <- (x_j cos - x_j+h sin, x_j+h cos + x_j sin) * factor
//
// with angle position * inv_freq[j], reduced in 64 bits. Q goes to query_out,
// K and V to their slots, K as stored into its page's bounds.
#include <math.h>

#include "paged.cuh"

namespace tla {

namespace {

constexpr int kThreads = 128;

// The sequence of row `row`, or -1: with offsets the last b with
// offsets[b] <= row, if the row lies before offsets[b + 1].
__device__ __forceinline__ int sequence_of(const int32_t* offsets, int batch, int row) {
  if (!offsets) return row;
  int lo = 0, hi = batch;  // offsets[lo] <= row < offsets[hi], once the ends are known to be so
  if (offsets[0] > row || offsets[batch] <= row) return -1;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (offsets[mid] <= row)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

template <typename CT>
__device__ __forceinline__ CT low_of(CT a, CT b) {
  return to_f32(b) < to_f32(a) ? b : a;
}
template <typename CT>
__device__ __forceinline__ CT high_of(CT a, CT b) {
  return to_f32(b) > to_f32(a) ? b : a;
}

// A block per row.
template <typename IO, typename CT>
__global__ void __launch_bounds__(kThreads)
    paged_append_kernel(PagedArgs p, const IO* __restrict__ qkv, const int32_t* __restrict__ offsets, int rows,
                        IO* __restrict__ query_out) {
  extern __shared__ float smem[];
  griddep_wait();
  griddep_launch_dependents();
  const LayerArgs& a = p.a;
  const int D = a.D, Hq = a.Hq, Hk = a.Hk, heads = Hq + 2 * Hk, half = a.rotary / 2;
  const int row = blockIdx.x;
  const int b = sequence_of(offsets, p.batch, row);
  if (b < 0) return;
  const int start = p.positions[b];
  const int pos = start < 0 || !offsets ? start
                  : static_cast<int>(min(start + (static_cast<long long>(row) - offsets[b]), 0x7fffffffLL));
  if (pos < 0 || pos >= p.capacity) {
    if (pos >= 0 && threadIdx.x == 0) report_error(a.error, TLA_ERR_POSITION);
    if (query_out)
      for (int i = threadIdx.x; i < Hq * D; i += kThreads)
        query_out[static_cast<int64_t>(row) * Hq * D + i] = from_f32<IO>(0.f);
    return;
  }
  float* x = smem;              // [heads * D]
  float* cs = smem + heads * D;  // [half] cos
  float* sn = cs + half;         // [half] sin
  const IO* src = qkv + static_cast<int64_t>(row) * heads * D;
  for (int i = threadIdx.x; i < heads * D; i += kThreads) x[i] = to_f32(src[i]);
  for (int j = threadIdx.x; j < half; j += kThreads) {
    float c = 1.f, s = 0.f;
    if (j < a.pair_count) rope_cos_sin(pos, a.inv_freq[j], &c, &s);
    cs[j] = c;
    sn[j] = s;
  }
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int h = warp; h < heads; h += kThreads / 32) {
    const float* w = h < Hq ? a.q_norm : h < Hq + Hk ? a.k_norm : nullptr;
    if (h < Hq + Hk ? w == nullptr : !a.v_norm) continue;
    float* v = x + h * D;
    float ss = 0.f;
    for (int d = lane; d < D; d += 32) ss += v[d] * v[d];
    const float inv_rms = 1.f / sqrtf(warp_sum(ss) / static_cast<float>(D) + a.rms_eps);
    for (int d = lane; d < D; d += 32) v[d] = v[d] * inv_rms * (w == nullptr ? 1.f : a.offset_rms ? 1.f + w[d] : w[d]);
  }
  __syncthreads();
  const int slot = pos & ((1 << p.page_shift) - 1);
  const int page = pool_page(p, b, pos >> p.page_shift);
  CT* key = static_cast<CT*>(p.key);
  CT* value = static_cast<CT*>(p.value);
  CT* bounds = static_cast<CT*>(p.bounds);
  for (int i = threadIdx.x; i < (Hq + Hk) * D; i += kThreads) {
    const int h = i / D, d = i - h * D;
    const float* v = x + h * D;
    float val = v[d];
    if (d < a.rotary) {
      const int j = d < half ? d : d - half;
      if (j < a.pair_count) {
        const float partner = d < half ? -v[d + half] : v[d - half];
        val = (val * cs[j] + partner * sn[j]) * a.attn_factor;
      }
    }
    if (h < Hq) {
      if (query_out) query_out[static_cast<int64_t>(row) * Hq * D + i] = from_f32<IO>(val);
    } else if (page >= 0) {
      const CT k = from_f32<CT>(val);
      key[pool_row(p, page, h - Hq, slot) + d] = k;
      if (bounds && !offsets) {  // one new token: its page's bounds right here
        CT* low = bounds + (static_cast<int64_t>(page) * Hk + (h - Hq)) * 2 * D + d;
        low[0] = slot == 0 ? k : low_of(low[0], k);
        low[D] = slot == 0 ? k : high_of(low[D], k);
      }
    }
  }
  if (page >= 0)
    for (int i = threadIdx.x; i < Hk * D; i += kThreads) {
      const int h = i / D;
      value[pool_row(p, page, h, slot) + (i - h * D)] = from_f32<CT>(x[(Hq + Hk) * D + i]);
    }
}

// Bounds of the pages that a chunk touched, from the keys as stored: the block
// of a page's first new row walks the page's new slots.
template <typename CT>
__global__ void __launch_bounds__(kThreads)
    paged_bounds_kernel(PagedArgs p, const int32_t* __restrict__ offsets, int rows) {
  griddep_wait();
  griddep_launch_dependents();
  const int D = p.a.D, Hk = p.a.Hk, row = blockIdx.x, mask = (1 << p.page_shift) - 1;
  const int b = sequence_of(offsets, p.batch, row);
  if (b < 0) return;
  const int start = p.positions[b];
  const long long done = static_cast<long long>(row) - offsets[b];
  if (start < 0 || start + done >= p.capacity) return;
  const int pos = start + static_cast<int>(done), slot = pos & mask;
  if (done != 0 && slot != 0) return;
  const int left = static_cast<int>(min(static_cast<long long>(min(offsets[b + 1], rows)) - row,
                                        static_cast<long long>(p.capacity) - pos));
  const int n = min(left, mask + 1 - slot);
  const int page = p.table[static_cast<int64_t>(b) * p.width + (pos >> p.page_shift)];
  if (static_cast<unsigned>(page) >= static_cast<unsigned>(p.page_count)) return;  // reported by the append
  const CT* key = static_cast<const CT*>(p.key);
  for (int i = threadIdx.x; i < Hk * D; i += kThreads) {
    const int h = i / D, d = i - h * D;
    CT* at = static_cast<CT*>(p.bounds) + (static_cast<int64_t>(page) * Hk + h) * 2 * D + d;
    const CT* k = key + pool_row(p, page, h, slot) + d;
    CT low = k[0], high = k[0];
    for (int s = 1; s < n; ++s) {
      const CT v = k[s * p.slot_stride];
      low = low_of(low, v);
      high = high_of(high, v);
    }
    at[0] = slot == 0 ? low : low_of(at[0], low);
    at[D] = slot == 0 ? high : high_of(at[D], high);
  }
}

template <typename IO, typename CT>
cudaError_t append_t(const PagedArgs& p, const void* qkv, const int32_t* offsets, int rows, void* query_out,
                     cudaStream_t stream) {
  const size_t smem = sizeof(float) * (static_cast<size_t>(p.a.Hq + 2 * p.a.Hk) * p.a.D + p.a.rotary);
  auto k = paged_append_kernel<IO, CT>;
  if (smem > 48 * 1024) {
    cudaError_t e = raise_smem_limit(reinterpret_cast<const void*>(k), static_cast<int>(smem));
    if (e != cudaSuccess) return e;
  }
  cudaError_t e = launch_pdl(k, rows, kThreads, smem, stream, p, static_cast<const IO*>(qkv), offsets, rows,
                             static_cast<IO*>(query_out));
  if (e != cudaSuccess || !p.bounds || !offsets) return e;
  return launch_pdl(paged_bounds_kernel<CT>, rows, kThreads, 0, stream, p, offsets, rows);
}

}  // namespace

cudaError_t launch_paged_append(const tla_paged* P, const PagedArgs& p, const void* qkv, const int32_t* offsets,
                                int rows, void* query_out, cudaStream_t stream) {
  if (P->io == kFp16) return append_t<__half, __half>(p, qkv, offsets, rows, query_out, stream);
  if (P->io == kBf16) return append_t<__nv_bfloat16, __nv_bfloat16>(p, qkv, offsets, rows, query_out, stream);
  if (P->kept == kFp16) return append_t<float, __half>(p, qkv, offsets, rows, query_out, stream);
  if (P->kept == kBf16) return append_t<float, __nv_bfloat16>(p, qkv, offsets, rows, query_out, stream);
  return append_t<float, float>(p, qkv, offsets, rows, query_out, stream);
}

}  // namespace tla
