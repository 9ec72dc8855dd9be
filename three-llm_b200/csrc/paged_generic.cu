// Paged decode for shapes that the tensor-core kernel does not take: any
// head_dim up to 256, float32 pages, pages of under 16 tokens, pools whose
// strides are not multiples of 16 bytes.
//
//   o = sum_t 2^(x_t - m) v_t / sum_t 2^(x_t - m),  x_t = log2(e) scale q.k_t
//
// A block of 4 warps takes up to 4 query heads of one kv head and one share of
// the sequence's tokens; a warp walks every fourth token with its lanes over
// the head's dimensions, so a row is one coalesced read that serves all four
// heads, and carries the running maximum, sum and output in registers. The
// warps' triples meet in shared memory, the blocks' in the workspace, where a
// second kernel joins them. Few sequences are split into more shares, so that
// about four blocks per SM stream at a time.
#include <math.h>

#include "paged.cuh"

namespace tla {

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kHeads = 4;     // query heads per block
constexpr int kMaxPer = 8;    // dimensions per lane: head_dim <= 256
constexpr int kMaxShares = 64;
constexpr float kLog2e = 1.4426950408889634f;

int head_chunks(const tla_paged* P) { return (P->base.G + kHeads - 1) / kHeads; }

int shares_of(const tla_paged* P, int batch) {
  const long long units = static_cast<long long>(batch) * P->base.Hk * head_chunks(P);
  const long long want = (4LL * P->base.ctx->sm_count + units - 1) / units;
  const long long most = (P->base.max_tokens + 127LL) / 128;
  const long long n = want < most ? want : most;
  return static_cast<int>(n < 1 ? 1 : n > kMaxShares ? kMaxShares : n);
}

template <typename IO>
__device__ __forceinline__ void store_out(IO* out, const IO* gate, int64_t i, float v) {
  if (gate) v = v * (1.f / (1.f + expf(-to_f32(gate[i]))));  // math.ts:271-273
  out[i] = from_f32<IO>(v);
}

template <typename IO, typename CT>
__global__ void __launch_bounds__(kThreads)
    paged_attend_kernel(PagedArgs p, const IO* __restrict__ query, const int32_t* __restrict__ pages, int count,
                        const IO* __restrict__ gate, IO* __restrict__ out, float* __restrict__ partial) {
  extern __shared__ float red[];  // [kWarps][kHeads][D + 2]
  griddep_wait();
  griddep_launch_dependents();
  const int D = p.a.D, G = p.a.G, Hk = p.a.Hk, Hq = p.a.Hq;
  const int chunks = (G + kHeads - 1) / kHeads;
  const int unit = blockIdx.y, kvh = unit / chunks, h0 = kvh * G + (unit % chunks) * kHeads;
  const int heads = min(kHeads, (kvh + 1) * G - h0);
  const int share = blockIdx.x, shares = gridDim.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int mask = (1 << p.page_shift) - 1;
  for (int b = blockIdx.z; b < p.batch; b += gridDim.z) {
    const int pos = p.positions[b];
    int lo, hi;
    if (!paged_range(p, pos, &lo, &hi) && pos >= 0 && threadIdx.x == 0) report_error(p.a.error, TLA_ERR_POSITION);
    const int32_t* list = pages ? pages + (static_cast<int64_t>(b) * Hk + kvh) * count : nullptr;
    int64_t n = hi - lo + 1;
    if (list) n = hi < 0 ? 0 : static_cast<int64_t>(list_length(p, list, count, hi >> p.page_shift, lane)) << p.page_shift;
    const int64_t begin = n * share / shares, end = n * (share + 1) / shares;
    float q[kHeads][kMaxPer], o[kHeads][kMaxPer], m[kHeads], l[kHeads];
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
      m[h] = -INFINITY;
      l[h] = 0.f;
#pragma unroll
      for (int e = 0; e < kMaxPer; ++e) {
        const int d = lane + 32 * e;
        q[h][e] = h < heads && d < D ? to_f32(query[(static_cast<int64_t>(b) * Hq + h0 + h) * D + d]) : 0.f;
        o[h][e] = 0.f;
      }
    }
    const float scale = p.a.attn_scale * kLog2e;
    for (int64_t j = begin + warp; j < end; j += kWarps) {
      const int t = list ? (list[j >> p.page_shift] << p.page_shift) + static_cast<int>(j & mask)
                         : lo + static_cast<int>(j);
      if (t < lo || t > hi) continue;  // (the same for the whole warp)
      const int page = pool_page(p, b, t >> p.page_shift);
      if (page < 0) continue;
      const int64_t row = pool_row(p, page, kvh, t & mask);
      const CT* k = static_cast<const CT*>(p.key) + row;
      const CT* v = static_cast<const CT*>(p.value) + row;
      float kf[kMaxPer], vf[kMaxPer];
#pragma unroll
      for (int e = 0; e < kMaxPer; ++e) {
        const int d = lane + 32 * e;
        kf[e] = d < D ? to_f32(k[d]) : 0.f;
        vf[e] = d < D ? to_f32(v[d]) : 0.f;
      }
#pragma unroll
      for (int h = 0; h < kHeads; ++h) {
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < kMaxPer; ++e) s += q[h][e] * kf[e];
        const float x = warp_sum(s) * scale;
        const float top = fmaxf(m[h], x), base = top == -INFINITY ? 0.f : top;
        const float keep = ex2(m[h] - base), w = ex2(x - base);
        m[h] = top;
        l[h] = l[h] * keep + w;
#pragma unroll
        for (int e = 0; e < kMaxPer; ++e) o[h][e] = o[h][e] * keep + w * vf[e];
      }
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
      float* r = red + (warp * kHeads + h) * (D + 2);
      if (lane == 0) {
        r[0] = m[h];
        r[1] = l[h];
      }
#pragma unroll
      for (int e = 0; e < kMaxPer; ++e)
        if (lane + 32 * e < D) r[2 + lane + 32 * e] = o[h][e];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < heads * D; i += kThreads) {
      const int h = i / D, d = i - h * D;
      float top = -INFINITY, sum = 0.f, acc = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, red[(w * kHeads + h) * (D + 2)]);
      if (top != -INFINITY) {
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float* r = red + (w * kHeads + h) * (D + 2);
          const float f = ex2(r[0] - top);
          sum += r[1] * f;
          acc += r[2 + d] * f;
        }
      }
      const int64_t row = static_cast<int64_t>(b) * Hq + h0 + h;
      if (shares > 1) {
        float* t = partial + (row * shares + share) * (D + 2);
        t[2 + d] = acc;
        if (d == 0) {
          t[0] = top;
          t[1] = sum;
        }
      } else {
        store_out(out, gate, row * D + d, sum > 0.f ? acc / sum : 0.f);
      }
    }
  }
}

// Joins the shares' triples; a block per output row.
template <typename IO>
__global__ void __launch_bounds__(kThreads)
    paged_join_kernel(const float* __restrict__ partial, int shares, int D, const IO* __restrict__ gate,
                      IO* __restrict__ out) {
  griddep_wait();
  griddep_launch_dependents();
  const int64_t row = blockIdx.x;
  const float* t = partial + row * shares * (D + 2);
  float top = -INFINITY;
  for (int s = 0; s < shares; ++s) top = fmaxf(top, t[s * (D + 2)]);
  for (int d = threadIdx.x; d < D; d += kThreads) {
    float sum = 0.f, acc = 0.f;
    if (top != -INFINITY) {
      for (int s = 0; s < shares; ++s) {
        const float f = ex2(t[s * (D + 2)] - top);
        sum += t[s * (D + 2) + 1] * f;
        acc += t[s * (D + 2) + 2 + d] * f;
      }
    }
    store_out(out, gate, row * D + d, sum > 0.f ? acc / sum : 0.f);
  }
}

template <typename IO, typename CT>
cudaError_t launch_t(const tla_paged* P, const PagedArgs& p, const void* query, const int32_t* pages, int count,
                     const void* gate, void* out, void* workspace, cudaStream_t stream) {
  const int shares = shares_of(P, p.batch), D = p.a.D;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(shares, p.a.Hk * head_chunks(P), p.batch < 65535 ? p.batch : 65535);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = sizeof(float) * kWarps * kHeads * (D + 2);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, paged_attend_kernel<IO, CT>, p, static_cast<const IO*>(query), pages, count,
                                     static_cast<const IO*>(gate), static_cast<IO*>(out),
                                     static_cast<float*>(workspace));
  if (e != cudaSuccess || shares == 1) return e;
  return launch_pdl(paged_join_kernel<IO>, static_cast<unsigned>(p.batch) * p.a.Hq, kThreads, 0, stream,
                    static_cast<const float*>(workspace), shares, D, static_cast<const IO*>(gate),
                    static_cast<IO*>(out));
}

}  // namespace

size_t paged_decode_generic_workspace(const tla_paged* P, int batch) {
  const int shares = shares_of(P, batch);
  return shares > 1 ? static_cast<size_t>(batch) * P->base.Hq * shares * (P->base.D + 2) * sizeof(float) : 0;
}

cudaError_t launch_paged_decode_generic(const tla_paged* P, const PagedArgs& p, const void* query,
                                        const int32_t* pages, int count, const void* gate, void* out, void* workspace,
                                        cudaStream_t stream) {
  if (P->io == kFp16) return launch_t<__half, __half>(P, p, query, pages, count, gate, out, workspace, stream);
  if (P->io == kBf16)
    return launch_t<__nv_bfloat16, __nv_bfloat16>(P, p, query, pages, count, gate, out, workspace, stream);
  if (P->kept == kFp16) return launch_t<float, __half>(P, p, query, pages, count, gate, out, workspace, stream);
  if (P->kept == kBf16)
    return launch_t<float, __nv_bfloat16>(P, p, query, pages, count, gate, out, workspace, stream);
  return launch_t<float, float>(P, p, query, pages, count, gate, out, workspace, stream);
}

}  // namespace tla
