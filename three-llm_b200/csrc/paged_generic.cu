// Paged decode for shapes that the tensor-core kernel does not take: float32
// pages, float32 activations over bfloat16 pages, pages of under 16 tokens
// (paged_rows_kernel); head_dims that are not multiples of 8 and pools whose
// strides are not multiples of 16 bytes (paged_attend_kernel).
//
//   o = sum_t 2^(x_t - m) v_t / sum_t 2^(x_t - m),  x_t = log2(e) scale q.k_t
//
// A block of 4 warps takes up to 4 query heads of one kv head and one share of
// the sequence's tokens; a row of the cache is read once for all four heads,
// and the running maximum, sum and output stay in registers. The warps' triples
// meet in shared memory, the blocks' in the workspace, where a second kernel
// joins them.
#include <math.h>

#include "paged.cuh"

namespace tla {

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kHeads = 4;     // query heads per block
constexpr int kMaxPer = 8;    // dimensions per lane: head_dim <= 256
constexpr int kMaxShares = 64;
constexpr int kBlocksPerSm = 3;
constexpr float kLog2e = 1.4426950408889634f;

int head_chunks(const tla_paged* P) { return (P->base.G + kHeads - 1) / kHeads; }

// Shares of a sequence's tokens: one wave of blocks where four shares or more
// fit it, else four waves of shorter ones, which even out ragged lengths.
int shares_of(const tla_paged* P, int batch) {
  const long long units = static_cast<long long>(batch) * P->base.Hk * head_chunks(P);
  const long long wave = static_cast<long long>(kBlocksPerSm) * P->base.ctx->sm_count;
  const long long want = wave / units >= 4 ? wave / units : 4 * wave / units;
  const long long most = (P->base.max_tokens + 127LL) / 128;
  const long long n = want < most ? want : most;
  return static_cast<int>(n < 1 ? 1 : n > kMaxShares ? kMaxShares : n);
}

// An output acc / sum times its gate; zero, whatever the gate holds, where no
// token took part. (gate and out may be the same memory: neither is declared
// __restrict__ in this file.)
template <typename IO>
__device__ __forceinline__ void store_out(IO* out, const IO* gate, int64_t i, float acc, float sum) {
  float v = sum != 0.f ? acc / sum : 0.f;
  if (gate && sum != 0.f) v = v * (1.f / (1.f + expf(-to_f32(gate[i]))));  // math.ts:271-273
  out[i] = from_f32<IO>(v);
}

// A block's output: its warps' triples [kWarps][kHeads][D + 2] joined, to the
// workspace, or where one block has all the tokens to the call's output.
template <typename IO>
__device__ __forceinline__ void join_warps(const float* red, int D, int heads, int64_t first_row, int share, int shares,
                                           const IO* gate, IO* out, float* __restrict__ partial) {
  for (int i = threadIdx.x; i < heads * D; i += kThreads) {
    const int h = i / D, d = i - h * D;
    float top = -INFINITY, sum = 0.f, acc = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, red[(w * kHeads + h) * (D + 2)]);
    const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float* r = red + (w * kHeads + h) * (D + 2);
      const float f = ex2(r[0] - base);
      sum += r[1] * f;
      acc += r[2 + d] * f;
    }
    const int64_t row = first_row + h;
    if (shares > 1) {
      float* t = partial + (row * shares + share) * (D + 2);
      t[2 + d] = acc;
      if (d == 0) {
        t[0] = top;
        t[1] = sum;
      }
    } else {
      store_out(out, gate, row * D + d, acc, sum);
    }
  }
}

template <typename IO, typename CT>
__global__ void __launch_bounds__(kThreads)
    paged_attend_kernel(PagedArgs p, const IO* __restrict__ query, const int32_t* __restrict__ pages, int count,
                        const IO* gate, IO* out, float* __restrict__ partial) {
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
    join_warps<IO>(red, D, heads, static_cast<int64_t>(b) * Hq + h0, share, shares, gate, out, partial);
  }
}

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int bytes) {  // bytes 0: zeroes
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// Two floats in one 64-bit register: a product or a sum of both is one instruction.
typedef unsigned long long Pair;
__device__ __forceinline__ Pair pair(float x, float y) {
  Pair v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y));
  return v;
}
__device__ __forceinline__ float2 halves(Pair v) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
  return f;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair v;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
  return v;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  Pair v;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}
// The elements of 16 bytes as pairs of floats.
__device__ __forceinline__ void unpack(const float4& u, Pair* x, float) {
  x[0] = pair(u.x, u.y);
  x[1] = pair(u.z, u.w);
}
__device__ __forceinline__ void unpack(const float4& u, Pair* x, __half) {
  const __half2* e = reinterpret_cast<const __half2*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(e[i]);
    x[i] = pair(f.x, f.y);
  }
}
__device__ __forceinline__ void unpack(const float4& u, Pair* x, __nv_bfloat16) {  // a float's upper half
  const uint32_t* e = reinterpret_cast<const uint32_t*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = pair(__uint_as_float(e[i] << 16), __uint_as_float(e[i] & 0xffff0000u));
}

// Rows on 16-byte boundaries, head_dim a multiple of 8 up to 16 LANES: LANES
// lanes hold a token, 16 of its dimensions each, so a warp works on 32 / LANES
// tokens at a time; the shuffles that add a score up leave each head's with the
// lanes that are to be its softmax's. Each group of lanes has a softmax of its
// own until the end, whose base follows the maximum only when that is kSlack
// ahead (weights up to 2^kSlack, in fp32): a rise makes the warp scale its
// outputs, and 32 maxima would rise nearly every step. A lane copies its pieces
// of the next kStages rows asynchronously to places that it alone reads, so that
// nothing waits for another lane; a row's page comes one step before its copy,
// its entry of a list two. CUDA-core products in fp32, two to an instruction: 8 x
// 4097 tokens, 32 / 8 heads of 64, float32 pages 34 us (3.9 TB/s), bfloat16
// pages 27 us, fp16 pages of 8 tokens 28 us (229, 299 and 300 us with a token
// per warp at a time).
constexpr float kSlack = 8.f;
constexpr int kStages = 4;
template <typename IO, typename CT, int LANES>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm)
    paged_rows_kernel(PagedArgs p, const IO* __restrict__ query, const int32_t* __restrict__ pages, int count,
                      const IO* gate, IO* out, float* __restrict__ partial) {
  constexpr int kPiece = 16 / sizeof(CT), kPieces = 16 / kPiece, kTokens = 32 / LANES, kStep = kWarps * kTokens;
  extern __shared__ float4 ring[];  // [kWarps][kStages][K, V][kPieces][32], then the warps' triples
  float* red = reinterpret_cast<float*>(ring);
  griddep_wait();
  griddep_launch_dependents();
  const int D = p.a.D, G = p.a.G, Hk = p.a.Hk, Hq = p.a.Hq;
  const int chunks = (G + kHeads - 1) / kHeads;
  const int unit = blockIdx.y, kvh = unit / chunks, h0 = kvh * G + (unit % chunks) * kHeads;
  const int heads = min(kHeads, (kvh + 1) * G - h0);
  const int share = blockIdx.x, shares = gridDim.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = lane / LANES, u = lane % LANES;
  const int shift = p.page_shift, mask = (1 << shift) - 1;
  const unsigned full = 0xffffffffu;
  const bool odd = u & 1, late = u & 2;  // the lane's head is 2 odd + late
  auto head_lane = [&](int h) { return lane - u + (h >> 1) + (h & 1) * 2; };
  const CT* const key = static_cast<const CT*>(p.key);
  const CT* const value = static_cast<const CT*>(p.value);
  float4* const own = ring + warp * (kStages * 2 * kPieces * 32) + lane;
  const uint32_t own_at = static_cast<uint32_t>(__cvta_generic_to_shared(own));
  int from[kPieces], size[kPieces];  // the lane's pieces of a row: elements, bytes (0 past its end)
#pragma unroll
  for (int c = 0; c < kPieces; ++c) {
    const int d = (c * LANES + u) * kPiece;
    from[c] = d < D ? d : 0;
    size[c] = d < D ? 16 : 0;
  }
  for (int b = blockIdx.z; b < p.batch; b += gridDim.z) {
    const int pos = p.positions[b];
    int lo, hi;
    if (!paged_range(p, pos, &lo, &hi) && pos >= 0 && threadIdx.x == 0) report_error(p.a.error, TLA_ERR_POSITION);
    const int32_t* list = pages ? pages + (static_cast<int64_t>(b) * Hk + kvh) * count : nullptr;
    int64_t n = hi - lo + 1;
    if (list) n = hi < 0 ? 0 : static_cast<int64_t>(list_length(p, list, count, hi >> shift, lane)) << shift;
    // (a token's number fits 32 bits without a sign: the list's pages are the sequence's own)
    const uint32_t begin = static_cast<uint32_t>(n * share / shares), end = static_cast<uint32_t>(n * (share + 1) / shares);
    const int steps = end > begin + warp * kTokens ? static_cast<int>((end - begin - warp * kTokens + kStep - 1) / kStep) : 0;
    const int32_t* const table = p.table + static_cast<int64_t>(b) * p.width;
    // The lanes' token of a step, j counting from the list's or the range's
    // first: its logical page (-1: none) and whether it takes part.
    auto logical = [&](uint32_t j) -> int { return j >= end ? -1 : list ? list[j >> shift] : static_cast<int>((lo + j) >> shift); };
    auto slot_of = [&](uint32_t j) -> int { return static_cast<int>(list ? j : lo + j) & mask; };
    auto takes = [&](uint32_t j, int at) -> bool {
      const int t = (at << shift) + slot_of(j);
      return at >= 0 && t >= lo && t <= hi;
    };
    uint32_t held = 0;  // a bit per stage: it holds a token
    auto copy = [&](int stage, uint32_t j, bool takes_part, int page) {
      const bool good = takes_part && static_cast<unsigned>(page) < static_cast<unsigned>(p.page_count);
      if (takes_part && !good) report_error(p.a.error, TLA_ERR_PAGE);
      held = good ? held | (1u << stage) : held & ~(1u << stage);
      const int64_t row = good ? pool_row(p, page, kvh, slot_of(j)) : 0;
      const CT* k = key + row;
      const CT* v = value + row;
#pragma unroll
      for (int c = 0; c < kPieces; ++c) {
        const int bytes = good ? size[c] : 0;
        copy16(own_at + ((stage * 2) * kPieces + c) * 512, k + from[c], bytes);
        copy16(own_at + ((stage * 2 + 1) * kPieces + c) * 512, v + from[c], bytes);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    uint32_t j = begin + warp * kTokens + group;
    bool takes_next;
    int entry = 0, after;  // step kStages's entry of the table, step kStages + 1's logical page
    {
      int at[kStages + 1], e[kStages + 1];
      bool part[kStages + 1];
#pragma unroll
      for (int s = 0; s <= kStages; ++s) at[s] = logical(j + s * kStep);
      after = logical(j + (kStages + 1) * kStep);
#pragma unroll
      for (int s = 0; s <= kStages; ++s) {
        part[s] = takes(j + s * kStep, at[s]);
        e[s] = part[s] ? table[at[s]] : 0;
      }
#pragma unroll
      for (int s = 0; s < kStages; ++s) copy(s, j + s * kStep, part[s], e[s]);
      takes_next = part[kStages];
      entry = e[kStages];
    }
    const float scale = p.a.attn_scale * kLog2e;
    Pair q[kHeads][8], o[kHeads][8];
    float m = -INFINITY, l = 0.f;  // of the lane's head
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int d = (2 * i / kPiece * LANES + u) * kPiece + 2 * i % kPiece;
        const IO* at = query + (static_cast<int64_t>(b) * Hq + h0 + h) * D + d;
        q[h][i] = h < heads && d < D ? pair(to_f32(at[0]) * scale, to_f32(at[1]) * scale) : pair(0.f, 0.f);
        o[h][i] = pair(0.f, 0.f);
      }
    }
    auto attend = [&](int stage) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
      const float4* k = own + stage * 2 * kPieces * 32;
      const float4* v = k + kPieces * 32;
      Pair xy[kHeads];
#pragma unroll
      for (int c = 0; c < kPieces; ++c) {
        Pair f[kPiece / 2];
        unpack(k[c * 32], f, CT());
#pragma unroll
        for (int h = 0; h < kHeads; ++h)
#pragma unroll
          for (int i = 0; i < kPiece / 2; ++i)
            xy[h] = c == 0 && i == 0 ? mul2(q[h][0], f[0]) : fma2(q[h][c * (kPiece / 2) + i], f[i], xy[h]);
      }
      float x[kHeads];
#pragma unroll
      for (int h = 0; h < kHeads; ++h) {
        const float2 f = halves(xy[h]);
        x[h] = f.x + f.y;
      }
      // each lane the sum of its own head
      const float y0 = (odd ? x[2] : x[0]) + __shfl_xor_sync(full, odd ? x[0] : x[2], 1);
      const float y1 = (odd ? x[3] : x[1]) + __shfl_xor_sync(full, odd ? x[1] : x[3], 1);
      float y = (late ? y1 : y0) + __shfl_xor_sync(full, late ? y0 : y1, 2);
#pragma unroll
      for (int w = 4; w < LANES; w <<= 1) y += __shfl_xor_sync(full, y, w);
      if (!(held >> stage & 1)) y = -INFINITY;
      if (__any_sync(full, y > m + kSlack)) {
        const float top = fmaxf(m, y), keep = top == -INFINITY ? 1.f : ex2(m - top);
        m = top;
        l *= keep;
#pragma unroll
        for (int h = 0; h < kHeads; ++h) {
          const float k_h = __shfl_sync(full, keep, head_lane(h));
#pragma unroll
          for (int i = 0; i < 8; ++i) o[h][i] = mul2(o[h][i], pair(k_h, k_h));
        }
      }
      y = y == -INFINITY ? 0.f : ex2(y - m);
      l += y;
#pragma unroll
      for (int h = 0; h < kHeads; ++h) x[h] = __shfl_sync(full, y, head_lane(h));
#pragma unroll
      for (int c = 0; c < kPieces; ++c) {
        Pair f[kPiece / 2];
        unpack(v[c * 32], f, CT());
#pragma unroll
        for (int h = 0; h < kHeads; ++h)
#pragma unroll
          for (int i = 0; i < kPiece / 2; ++i)
            o[h][c * (kPiece / 2) + i] = fma2(pair(x[h], x[h]), f[i], o[h][c * (kPiece / 2) + i]);
      }
      copy(stage, j + kStages * kStep, takes_next, entry);
      takes_next = takes(j + (kStages + 1) * kStep, after);
      entry = takes_next ? table[after] : 0;
      after = logical(j + (kStages + 2) * kStep);
      j += kStep;
    };
    for (int step = 0; step < steps; step += kStages) {
#pragma unroll
      for (int s = 0; s < kStages; ++s)
        if (step + s < steps) attend(s);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    // the groups of the warp, then the warps
    float top = m;
#pragma unroll
    for (int w = LANES; w < 32; w <<= 1) top = fmaxf(top, __shfl_xor_sync(full, top, w));
    const float keep = top == -INFINITY ? 1.f : ex2(m - top);
    l *= keep;
#pragma unroll
    for (int w = LANES; w < 32; w <<= 1) l += __shfl_xor_sync(full, l, w);
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
      const float k_h = __shfl_sync(full, keep, head_lane(h));
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float2 f = halves(mul2(o[h][i], pair(k_h, k_h)));
#pragma unroll
        for (int w = LANES; w < 32; w <<= 1) {
          f.x += __shfl_xor_sync(full, f.x, w);
          f.y += __shfl_xor_sync(full, f.y, w);
        }
        o[h][i] = pair(f.x, f.y);
      }
    }
    __syncthreads();  // every warp is done with its ring, which the triples overwrite
    if (group == 0) {
#pragma unroll
      for (int h = 0; h < kHeads; ++h) {
        float* r = red + (warp * kHeads + h) * (D + 2);
        if (lane == head_lane(h)) {
          r[0] = top;
          r[1] = l;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int d = (2 * i / kPiece * LANES + u) * kPiece + 2 * i % kPiece;
          if (d < D) *reinterpret_cast<float2*>(r + 2 + d) = halves(o[h][i]);
        }
      }
    }
    __syncthreads();
    join_warps<IO>(red, D, heads, static_cast<int64_t>(b) * Hq + h0, share, shares, gate, out, partial);
    __syncthreads();
  }
}

// Joins the shares' triples; a block per output row.
template <typename IO>
__global__ void __launch_bounds__(kThreads)
    paged_join_kernel(const float* __restrict__ partial, int shares, int D, const IO* gate, IO* out) {
  griddep_wait();
  griddep_launch_dependents();
  const int64_t row = blockIdx.x;
  const float* t = partial + row * shares * (D + 2);
  float top = -INFINITY;
  for (int s = 0; s < shares; ++s) top = fmaxf(top, t[s * (D + 2)]);
  const float base = top == -INFINITY ? 0.f : top;
  for (int d = threadIdx.x; d < D; d += kThreads) {
    float sum = 0.f, acc = 0.f;
    for (int s = 0; s < shares; ++s) {
      const float f = ex2(t[s * (D + 2)] - base);
      sum += t[s * (D + 2) + 1] * f;
      acc += t[s * (D + 2) + 2 + d] * f;
    }
    store_out(out, gate, row * D + d, acc, sum);
  }
}

template <typename IO, typename CT>
cudaError_t launch_t(const tla_paged* P, const PagedArgs& p, const void* query, const int32_t* pages, int count,
                     const void* gate, void* out, void* workspace, cudaStream_t stream) {
  const int shares = shares_of(P, p.batch), D = p.a.D;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(shares, p.a.Hk * head_chunks(P), p.batch < 65535 ? p.batch : 65535);
  cfg.blockDim = dim3(kThreads);
  const size_t triples = sizeof(float) * kWarps * kHeads * (D + 2);
  const size_t ring = P->wide ? sizeof(CT) * kWarps * kStages * 2 * 16 * 32 : 0;
  cfg.dynamicSmemBytes = triples > ring ? triples : ring;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  auto kernel = !P->wide   ? paged_attend_kernel<IO, CT>
                : D <= 64  ? paged_rows_kernel<IO, CT, 4>
                : D <= 128 ? paged_rows_kernel<IO, CT, 8>
                           : paged_rows_kernel<IO, CT, 16>;
  cudaError_t e = cfg.dynamicSmemBytes > 48 * 1024
                      ? raise_smem_limit(reinterpret_cast<const void*>(kernel), static_cast<int>(cfg.dynamicSmemBytes))
                      : cudaSuccess;
  if (e != cudaSuccess) return e;
  e = cudaLaunchKernelEx(&cfg, kernel, p, static_cast<const IO*>(query), pages, count,
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
