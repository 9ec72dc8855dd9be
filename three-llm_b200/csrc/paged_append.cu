// Appending rows of [Q | K | V] to a paged cache (the copy-KV and query
// kernels of TSLAttention, packages/three-llm/src/tsl/TSLAttention.ts:252-304,
// with the slot looked up in a page table):
//
//   x <- x / sqrt(mean(x^2) + eps) * w          QK-norm (vNorm: w = 1)
//   (x_j, x_j+h) <- (x_j cos - x_j+h sin, x_j+h cos + x_j sin) * factor
//
// with angle position * inv_freq[j], reduced in 64 bits. Q goes to query_out,
// K and V to their slots, K as stored into its page's bounds.
//
// Every value is read and written once, so memory bounds long calls: 20,500 rows
// of 16 ragged chunks with bounds, 48 heads of 128, bfloat16, QK-norm, in 93 us
// (0.86 of a copy's rate, issue slots 64% busy); one new token each of 64
// sequences takes 2.6 us, a chain of offsets, position, table entry and row.
#include <math.h>

#include <type_traits>

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

// The same by a whole warp, 32 offsets at a time: two rounds of loads for up to
// 1024 sequences where the search above takes ten.
__device__ __forceinline__ int sequence_of_warp(const int32_t* offsets, int batch, int row, int lane) {
  if (!offsets) return row;
  int lo = 0, n = batch + 1;  // the answer is the last of [lo, lo + n) that is <= row
  while (n > 1) {
    const int step = (n + 31) / 32, at = lo + lane * step;
    const unsigned low = __ballot_sync(0xffffffffu, at < lo + n && offsets[min(at, batch)] <= row);
    if (low == 0) return -1;  // (only possible in the first round: row lies before offsets[0])
    const int last = 31 - __clz(low);
    n = min(step, lo + n - (lo + last * step));
    lo += last * step;
  }
  // (offsets out of order may lead anywhere: what counts is that the row lies in the sequence found)
  return lo < batch && offsets[lo] <= row && row < offsets[lo + 1] ? lo : -1;
}

// The smaller and the larger of two; what is no number gives way to a number.
template <typename CT>
__device__ __forceinline__ CT low_of(CT a, CT b) {
  const float x = to_f32(a), y = to_f32(b);
  return y < x || x != x ? b : a;
}
template <typename CT>
__device__ __forceinline__ CT high_of(CT a, CT b) {
  const float x = to_f32(a), y = to_f32(b);
  return y > x || x != x ? b : a;
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
        CT* low = bounds + bounds_row(p, page, h - Hq, D) + d;
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

// Four neighbouring elements, as loaded and as floats.
template <typename T>
struct Raw4 {
  uint2 u;
};
template <>
struct Raw4<float> {
  float4 u;
};
template <typename T>
__device__ __forceinline__ Raw4<T> raw4(const T* p) {
  return *reinterpret_cast<const Raw4<T>*>(p);
}
__device__ __forceinline__ float4 floats(const Raw4<float>& r) { return r.u; }
__device__ __forceinline__ float4 floats(const Raw4<__half>& r) {
  const uint2 u = r.u;
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&u.x));
  const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
  return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ float4 floats(const Raw4<__nv_bfloat16>& r) {
  const uint2 u = r.u;
  return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                     __uint_as_float(u.y & 0xffff0000u));
}
template <typename T>
__device__ __forceinline__ void put4(T* p, Raw4<T> v) {
  *reinterpret_cast<Raw4<T>*>(p) = v;
}
// Four floats rounded to T.
template <typename T>
__device__ __forceinline__ Raw4<T> pack4(float4 v) {
  if constexpr (sizeof(T) == 4) {
    return {v};
  } else if constexpr (std::is_same<T, __half>::value) {
    return {make_uint2(pack_half2(v.x, v.y), pack_half2(v.z, v.w))};
  } else {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
    return {make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b))};
  }
}
template <typename T>
__device__ __forceinline__ void store4(T* p, float4 v) {
  put4(p, pack4<T>(v));
}
// What was loaded, stored without a detour where the types are the same.
template <typename T>
__device__ __forceinline__ void put_same(T* p, Raw4<T> v) {
  put4(p, v);
}
template <typename T, typename U>
__device__ __forceinline__ void put_same(T* p, Raw4<U> v) {
  store4(p, floats(v));
}

// The same of pairs and of four.
template <typename P>
__device__ __forceinline__ uint32_t low_pair(uint32_t a, uint32_t b) {
  const P v = __hmin2(*reinterpret_cast<P*>(&a), *reinterpret_cast<P*>(&b));
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <typename P>
__device__ __forceinline__ uint32_t high_pair(uint32_t a, uint32_t b) {
  const P v = __hmax2(*reinterpret_cast<P*>(&a), *reinterpret_cast<P*>(&b));
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <typename T>
__device__ __forceinline__ Raw4<T> low4(Raw4<T> a, Raw4<T> b) {
  if constexpr (sizeof(T) == 4) {
    return {make_float4(fminf(a.u.x, b.u.x), fminf(a.u.y, b.u.y), fminf(a.u.z, b.u.z), fminf(a.u.w, b.u.w))};
  } else {
    using P = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    return {make_uint2(low_pair<P>(a.u.x, b.u.x), low_pair<P>(a.u.y, b.u.y))};
  }
}
template <typename T>
__device__ __forceinline__ Raw4<T> high4(Raw4<T> a, Raw4<T> b) {
  if constexpr (sizeof(T) == 4) {
    return {make_float4(fmaxf(a.u.x, b.u.x), fmaxf(a.u.y, b.u.y), fmaxf(a.u.z, b.u.z), fmaxf(a.u.w, b.u.w))};
  } else {
    using P = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    return {make_uint2(high_pair<P>(a.u.x, b.u.x), high_pair<P>(a.u.y, b.u.y))};
  }
}
template <typename T>
__device__ __forceinline__ Raw4<T> lane_xor(Raw4<T> v, int o) {
  if constexpr (sizeof(T) == 4)
    return {make_float4(__shfl_xor_sync(0xffffffffu, v.u.x, o), __shfl_xor_sync(0xffffffffu, v.u.y, o),
                        __shfl_xor_sync(0xffffffffu, v.u.z, o), __shfl_xor_sync(0xffffffffu, v.u.w, o))};
  else
    return {make_uint2(__shfl_xor_sync(0xffffffffu, v.u.x, o), __shfl_xor_sync(0xffffffffu, v.u.y, o))};
}

// head_dim and the rotary dimensions multiples of 8: D / 8 lanes hold a head (D
// is head_dim, or where !EXACT 128 or 256, its last lanes idle), each the four
// rotation pairs 4 l .. 4 l + 3 (both elements, so that no lane needs another's;
// dimensions past the rotary ones pair up among themselves and stay). `parts`
// warps share a row's heads, so that few rows still fill the GPU; a warp forms
// the row's cosines and sines once, one or two per lane, and hands them out by
// shuffles (at 256 each lane its own four). Without `keys` the row's keys are
// left to the blocks that go by pages. `unit`: the warp's (row, part).
// TURNED: the rotation turns every dimension.
template <typename IO, typename CT, int D, bool EXACT, bool TURNED>
__device__ __forceinline__ void append_rows(const PagedArgs& p, const IO* __restrict__ qkv,
                                            const int32_t* __restrict__ offsets, int rows,
                                            IO* __restrict__ query_out, int parts, int part_heads, bool keys,
                                            int64_t unit) {
  constexpr int kLanes = D / 8, kPer = 32 / kLanes;  // lanes per head, heads per warp-wide load
  constexpr int kLoads = sizeof(IO) == 2 ? 4 : 2;    // warp-wide loads in flight
  const unsigned full = 0xffffffffu;
  const LayerArgs& a = p.a;
  const int Hq = a.Hq, Hk = a.Hk, heads = Hq + 2 * Hk, half = a.rotary / 2;
  const int lane = threadIdx.x & 31, group = lane / kLanes, i0 = 4 * (lane % kLanes);
  const int hd = EXACT ? D : a.D;
  const bool on = EXACT || 2 * i0 < hd;
  const int row = static_cast<int>(unit / parts), part = static_cast<int>(unit % parts);
  // the first elements of the lane's four pairs, and their partners
  const int d0 = i0 < half ? i0 : a.rotary + i0 - half;
  const int d1 = d0 + (i0 < half ? half : (hd - a.rotary) / 2);
  if (row >= rows) return;
  // the part's heads: queries, keys (or none), values
  const int k_heads = keys ? Hk : 0, h_begin = part * part_heads;
  const int h_end = min(Hq + k_heads + Hk, h_begin + part_heads);
  const IO* src = qkv + static_cast<int64_t>(row) * heads * hd;
  const int b = sequence_of_warp(offsets, p.batch, row, lane);
  if (b < 0) return;
  const int start = p.positions[b];
  const int pos = start < 0 || !offsets ? start
                  : static_cast<int>(min(start + (static_cast<long long>(row) - offsets[b]), 0x7fffffffLL));
  if (pos < 0 || pos >= p.capacity) {
    if (pos >= 0 && lane == 0) report_error(a.error, TLA_ERR_POSITION);
    if (query_out)
      for (int h = h_begin + group; h < min(h_end, Hq); h += kPer) {
        IO* q = query_out + (static_cast<int64_t>(row) * Hq + h) * hd;
        if (!on) continue;
        store4(q + d0, make_float4(0.f, 0.f, 0.f, 0.f));
        store4(q + d1, make_float4(0.f, 0.f, 0.f, 0.f));
      }
    return;
  }
  const int slot = pos & ((1 << p.page_shift) - 1);
  // (a part with queries only does not need the page)
  const int page = h_end > Hq ? pool_page(p, b, pos >> p.page_shift) : -1;
  const int turned = i0 < half ? min(a.pair_count, half) - i0 : 0;  // of this lane's pairs, those before this one
  float cos4[4], sin4[4];
  if (h_begin < Hq + k_heads) {
    float c0 = 1.f, s0 = 0.f, c1 = 1.f, s1 = 0.f;
    if (D < 256 && lane < min(a.pair_count, half)) rope_cos_sin(pos, a.inv_freq[lane], &c0, &s0);
    if (D == 128 && lane + 32 < min(a.pair_count, half)) rope_cos_sin(pos, a.inv_freq[lane + 32], &c1, &s1);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int src_lane = (i0 + e) & 31;
      float c = 1.f, s = 0.f;
      if (D == 256) {
        if (e < turned) rope_cos_sin(pos, a.inv_freq[i0 + e], &c, &s);
      } else {
        c = __shfl_sync(full, c0, src_lane);
        s = __shfl_sync(full, s0, src_lane);
      }
      if (D == 128) {
        const float ch = __shfl_sync(full, c1, src_lane), sh = __shfl_sync(full, s1, src_lane);
        if (i0 + e >= 32) {
          c = ch;
          s = sh;
        }
      }
      cos4[e] = e < turned ? c * a.attn_factor : 1.f;
      sin4[e] = e < turned ? s * a.attn_factor : 0.f;
    }
  }
  // Heads [from, to) of one kind: 0 queries, 1 keys, 2 values.
  auto heads_of = [&](auto kind, int from, int to, const float* w, bool norm) {
    constexpr int kKind = decltype(kind)::value;
    if (from >= to) return;
    if (kKind == 0 ? query_out == nullptr : page < 0) return;
    // The norm's weights folded into the rotation: (x, y) of a pair becomes
    // r (x xc - y ys, y yc + x xs), r = 1 / rms.
    float xc[4], xs[4], yc[4], ys[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float add = a.offset_rms ? 1.f : 0.f;
      const float wx = w == nullptr || !on ? 1.f : add + w[d0 + e], wy = w == nullptr || !on ? 1.f : add + w[d1 + e];
      xc[e] = kKind == 2 ? 1.f : wx * cos4[e];
      xs[e] = kKind == 2 ? 0.f : wx * sin4[e];
      yc[e] = kKind == 2 ? 1.f : wy * cos4[e];
      ys[e] = kKind == 2 ? 0.f : wy * sin4[e];
    }
    const IO* in = src + (from + group) * hd;
    IO* q = kKind == 0 ? query_out + (static_cast<int64_t>(row) * Hq + from + group) * hd : nullptr;
    CT* kv = kKind == 0 ? nullptr : static_cast<CT*>(kKind == 1 ? p.key : p.value) + pool_row(p, page, 0, slot);
    for (int h0 = from + group; h0 - group < to; h0 += kLoads * kPer, in += kLoads * kPer * hd, q += kLoads * kPer * hd) {
      Raw4<IO> lo[kLoads], hi[kLoads];
#pragma unroll
      for (int c = 0; c < kLoads; ++c) {
        const bool in_part = on && h0 + c * kPer < to;
        lo[c] = in_part ? raw4(in + c * kPer * hd + d0) : Raw4<IO>{};
        hi[c] = in_part ? raw4(in + c * kPer * hd + d1) : Raw4<IO>{};
      }
      float r[kLoads];
      if (norm) {  // math.ts:78-97; the loads' sums go through the shuffles side by side
#pragma unroll
        for (int c = 0; c < kLoads; ++c) {
          const float4 x = floats(lo[c]), y = floats(hi[c]);
          r[c] = x.x * x.x + x.y * x.y + x.z * x.z + x.w * x.w + y.x * y.x + y.y * y.y + y.z * y.z + y.w * y.w;
        }
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1)
#pragma unroll
          for (int c = 0; c < kLoads; ++c) r[c] += __shfl_xor_sync(full, r[c], o);
#pragma unroll
        for (int c = 0; c < kLoads; ++c) r[c] = rsqrtf(r[c] * (1.f / hd) + a.rms_eps);  // (2 ulp)
      }
#pragma unroll
      for (int c = 0; c < kLoads; ++c) {
        float4 x = floats(lo[c]), y = floats(hi[c]);
        if (norm) {
          x = make_float4(x.x * r[c], x.y * r[c], x.z * r[c], x.w * r[c]);
          y = make_float4(y.x * r[c], y.y * r[c], y.z * r[c], y.w * r[c]);
        }
        if (kKind < 2) {  // RoPE, math.ts:134-147
          // (a dimension that stays takes nothing from its partner, not even 0 times an infinity)
          const float4 u = x, v = y;
          const auto from = [&](int e, float partner) { return TURNED || e < turned ? partner : 0.f; };
          x = make_float4(u.x * xc[0] - from(0, v.x) * ys[0], u.y * xc[1] - from(1, v.y) * ys[1],
                          u.z * xc[2] - from(2, v.z) * ys[2], u.w * xc[3] - from(3, v.w) * ys[3]);
          y = make_float4(v.x * yc[0] + from(0, u.x) * xs[0], v.y * yc[1] + from(1, u.y) * xs[1],
                          v.z * yc[2] + from(2, u.z) * xs[2], v.w * yc[3] + from(3, u.w) * xs[3]);
        }
        const int h = h0 + c * kPer;
        if (h >= to || !on) continue;
        if (kKind == 0) {
          store4(q + c * kPer * hd + d0, x);
          store4(q + c * kPer * hd + d1, y);
        } else {
          const int kvh = h - Hq - (kKind == 1 ? 0 : Hk);
          CT* at = kv + kvh * p.head_stride;
          if (kKind == 2 && !norm) {  // values stay as they are
            put_same(at + d0, lo[c]);
            put_same(at + d1, hi[c]);
          } else {
            store4(at + d0, x);
            store4(at + d1, y);
          }
          if (kKind == 1 && p.bounds && !offsets) {  // one new token: its page's bounds right here
            CT* low = static_cast<CT*>(p.bounds) + bounds_row(p, page, kvh, hd);
            CT* high = low + hd;
            const Raw4<CT> k0 = pack4<CT>(x), k1 = pack4<CT>(y);
            put4(low + d0, slot == 0 ? k0 : low4<CT>(raw4(low + d0), k0));
            put4(low + d1, slot == 0 ? k1 : low4<CT>(raw4(low + d1), k1));
            put4(high + d0, slot == 0 ? k0 : high4<CT>(raw4(high + d0), k0));
            put4(high + d1, slot == 0 ? k1 : high4<CT>(raw4(high + d1), k1));
          }
        }
      }
    }
  };
  heads_of(std::integral_constant<int, 0>(), h_begin, min(h_end, Hq), a.q_norm, a.q_norm != nullptr);
  heads_of(std::integral_constant<int, 1>(), max(h_begin, Hq), min(h_end, Hq + k_heads), a.k_norm, a.k_norm != nullptr);
  const int skipped = Hk - k_heads;
  heads_of(std::integral_constant<int, 2>(), max(h_begin + skipped, Hq + Hk), h_end + skipped, nullptr, a.v_norm != 0);
}

// Pages that sequence b's chunk goes to (0: none), its rows cut off where the
// positions or the rows end.
struct Chunk {
  int row, start, n;
};
__device__ __forceinline__ Chunk chunk_of(const PagedArgs& p, const int32_t* offsets, int rows, int b) {
  const int start = p.positions[b], row = offsets[b];
  const long long end = min(static_cast<long long>(offsets[b + 1]), static_cast<long long>(rows));
  if (start < 0 || start >= p.capacity || row < 0 || end <= row) return {0, 0, 0};
  return {row, start, static_cast<int>(min(end - row, static_cast<long long>(p.capacity) - start))};
}
__device__ __forceinline__ int pages_of(const PagedArgs& p, const Chunk& c) {
  return c.n == 0 ? 0 : ((c.start + c.n - 1) >> p.page_shift) - (c.start >> p.page_shift) + 1;
}

// The touched page of a launch that a block works on: page `want` of all the
// chunks' touched pages in order, found by a scan of the sequences' page
// counts. False when there are fewer.
template <int kBlock>
__device__ __forceinline__ bool find_page(const PagedArgs& p, const int32_t* offsets, int rows, int want, int* b_out,
                                          int* nth) {
  __shared__ int sums[kBlock / 32];
  __shared__ int found[2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int before = 0;
  if (tid == 0) found[0] = -1;
  for (int base = 0; base < p.batch; base += kBlock) {
    const int b = base + tid;
    const int n = b < p.batch ? pages_of(p, chunk_of(p, offsets, rows, b)) : 0;
    int scan = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, scan, o);
      if (lane >= o) scan += v;
    }
    if (lane == 31) sums[warp] = scan;
    __syncthreads();
    int all = 0;
    for (int i = 0; i < kBlock / 32; ++i) {
      if (i < warp) scan += sums[i];
      all += sums[i];
    }
    scan += before;  // pages up to and with sequence b's
    if (n > 0 && want < scan && want >= scan - n) {
      found[0] = b;
      found[1] = want - (scan - n);
    }
    before += all;
    __syncthreads();
    if (found[0] >= 0) break;
  }
  *b_out = found[0];
  *nth = found[1];
  return found[0] >= 0;
}

// The keys of one touched page and `heads` kv heads (1, 2, 4 or 8), and the
// page's bounds: 8 / heads warps per head keep the smallest and largest keys
// in registers while they rotate and store them. The cosines and
// sines of kPageSlots slots are formed in shared memory at a time, from those
// of the first slot and a table of those of 0 .. kPageSlots - 1 steps:
// cos(a + b) = cos a cos b - sin a sin b and its like add three roundings and
// spare 31 of 32 evaluations, which with few rows per block would bound it.
constexpr int kPageThreads = 256;
template <typename IO, typename CT, int D, bool EXACT, bool TURNED>
__device__ __forceinline__ void append_page(const PagedArgs& p, const IO* __restrict__ qkv,
                                            const int32_t* __restrict__ offsets, int rows, int heads, int unit) {
  constexpr int kLanes = D / 8, kPer = 32 / kLanes, kWarps = kPageThreads / 32;
  constexpr int kLoads = 4;  // warp-wide loads in flight
  constexpr int kPageSlots = D == 256 ? kTurnSteps / 2 : kTurnSteps;
  const unsigned full = 0xffffffffu;
  __shared__ float2 base_s[D / 2];
  __shared__ float2 turn_s[kPageSlots][D / 2];
  __shared__ __align__(16) float join_s[kWarps][2][D];
  const LayerArgs& a = p.a;
  const int Hk = a.Hk, half = a.rotary / 2, pairs = min(a.pair_count, half);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, group = lane / kLanes, i0 = 4 * (lane % kLanes);
  const int hd = EXACT ? D : a.D;
  const bool on = EXACT || 2 * i0 < hd;
  const int groups = (Hk + heads - 1) / heads;
  int b, nth;
  if (!find_page<kPageThreads>(p, offsets, rows, unit / groups, &b, &nth)) return;
  const Chunk c = chunk_of(p, offsets, rows, b);
  const int index = (c.start >> p.page_shift) + nth, size = 1 << p.page_shift;
  const int page = pool_page(p, b, index);
  if (page < 0) return;
  const int64_t from = static_cast<int64_t>(index) << p.page_shift;  // the position of slot 0
  const int begin = static_cast<int>(max(static_cast<int64_t>(0), c.start - from));
  const int end = static_cast<int>(min(static_cast<int64_t>(size), c.start + static_cast<int64_t>(c.n) - from));
  const int64_t row0 = c.row + from - c.start;  // the row of slot 0 (of slots >= begin)
  const int d0 = i0 < half ? i0 : a.rotary + i0 - half;
  const int d1 = d0 + (i0 < half ? half : (hd - a.rotary) / 2);
  const int shares = kWarps / heads, share = warp / heads;  // warps per head, and this one's place
  const int kvh = unit % groups * heads + warp % heads;
  const int row_size = (a.Hq + 2 * Hk) * hd;
  Raw4<CT> low0 = pack4<CT>(make_float4(INFINITY, INFINITY, INFINITY, INFINITY)), low1 = low0;
  Raw4<CT> high0 = pack4<CT>(make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY)), high1 = high0;
  for (int s0 = begin; s0 < end; s0 += kPageSlots) {
    const int slots = min(kPageSlots, end - s0);
    __syncthreads();
    for (int j = tid; j < pairs; j += kPageThreads) {
      float cs, sn;
      rope_cos_sin(static_cast<int>(from + s0), a.inv_freq[j], &cs, &sn);
      base_s[j] = make_float2(cs * a.attn_factor, sn * a.attn_factor);
    }
    __syncthreads();
    for (int i = tid; i < slots * (D / 2); i += kPageThreads) {
      const int s = i / (D / 2), j = i - s * (D / 2);
      float2 v = make_float2(1.f, 0.f);
      if (j < pairs) {
        const float2 x = base_s[j], y = p.turns[s * half + j];
        v = make_float2(x.x * y.x - x.y * y.y, x.y * y.x + x.x * y.y);
      }
      turn_s[s][j] = v;
    }
    __syncthreads();
    if (kvh >= Hk) continue;
    const IO* in = qkv + (row0 + s0) * row_size + (a.Hq + kvh) * hd;
    CT* out = static_cast<CT*>(p.key) + pool_row(p, page, kvh, s0);
    for (int s1 = share * kPer + group; s1 - group < slots; s1 += shares * kPer * kLoads) {
      Raw4<IO> lo[kLoads], hi[kLoads];
#pragma unroll
      for (int k = 0; k < kLoads; ++k) {
        const int s = s1 + k * shares * kPer;
        const bool held = on && s < slots && TLA_IN_BOUNDS(row0 + s0 + s, rows, a.error);
        lo[k] = held ? raw4(in + static_cast<int64_t>(s) * row_size + d0) : Raw4<IO>{};
        hi[k] = held ? raw4(in + static_cast<int64_t>(s) * row_size + d1) : Raw4<IO>{};
      }
#pragma unroll
      for (int k = 0; k < kLoads; ++k) {
        const int s = s1 + k * shares * kPer;
        const float4 xf = floats(lo[k]), yf = floats(hi[k]);
        float x[4] = {xf.x, xf.y, xf.z, xf.w}, y[4] = {yf.x, yf.y, yf.z, yf.w};
        if (a.k_norm) {  // math.ts:78-97
          float ss = 0.f;
#pragma unroll
          for (int e = 0; e < 4; ++e) ss += x[e] * x[e] + y[e] * y[e];
#pragma unroll
          for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(full, ss, o);
          const float r = rsqrtf(ss * (1.f / hd) + a.rms_eps);  // (2 ulp)
          const float add = a.offset_rms ? 1.f : 0.f;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            x[e] *= r * (on ? add + __ldg(a.k_norm + d0 + e) : 0.f);
            y[e] *= r * (on ? add + __ldg(a.k_norm + d1 + e) : 0.f);
          }
        }
        if (s >= slots || !on) continue;
        if (i0 < half) {  // RoPE, math.ts:134-147
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 t = turn_s[s][i0 + e];
            const bool turned = TURNED || i0 + e < pairs;  // (else nothing comes over, not even 0 times an infinity)
            const float u = x[e] * t.x - (turned ? y[e] : 0.f) * t.y;
            y[e] = y[e] * t.x + (turned ? x[e] : 0.f) * t.y;
            x[e] = u;
          }
        }
        const Raw4<CT> k0 = pack4<CT>(make_float4(x[0], x[1], x[2], x[3]));
        const Raw4<CT> k1 = pack4<CT>(make_float4(y[0], y[1], y[2], y[3]));
        put4(out + s * p.slot_stride + d0, k0);
        put4(out + s * p.slot_stride + d1, k1);
        low0 = low4<CT>(low0, k0);
        low1 = low4<CT>(low1, k1);
        high0 = high4<CT>(high0, k0);
        high1 = high4<CT>(high1, k1);
      }
    }
  }
  // across the lanes' slots, then the warps of a head
#pragma unroll
  for (int o = kLanes; o < 32; o <<= 1) {
    low0 = low4<CT>(low0, lane_xor<CT>(low0, o));
    low1 = low4<CT>(low1, lane_xor<CT>(low1, o));
    high0 = high4<CT>(high0, lane_xor<CT>(high0, o));
    high1 = high4<CT>(high1, lane_xor<CT>(high1, o));
  }
  if (group == 0 && on) {
    *reinterpret_cast<float4*>(&join_s[warp][0][d0]) = floats(low0);
    *reinterpret_cast<float4*>(&join_s[warp][0][d1]) = floats(low1);
    *reinterpret_cast<float4*>(&join_s[warp][1][d0]) = floats(high0);
    *reinterpret_cast<float4*>(&join_s[warp][1][d1]) = floats(high1);
  }
  __syncthreads();
  for (int i = tid; i < heads * 2 * hd; i += kPageThreads) {  // [head][low, high][d]
    const int h = i / (2 * hd), at = i - h * 2 * hd, head = unit % groups * heads + h;
    const bool is_low = at < hd;
    const int e = is_low ? at : at - hd;
    if (head >= Hk) continue;
    float v = join_s[h][is_low ? 0 : 1][e];
    for (int k = 1; k < shares; ++k) {
      const float u = join_s[h + k * heads][is_low ? 0 : 1][e];
      v = (is_low ? u < v : u > v) ? u : v;
    }
    CT* to = static_cast<CT*>(p.bounds) + bounds_row(p, page, head, hd) + at;
    if (begin > 0) v = is_low ? low_of(to_f32(to[0]), v) : high_of(to_f32(to[0]), v);
    to[0] = from_f32<CT>(v);
  }
}

// Rows only.
template <typename IO, typename CT, int D, bool EXACT, bool TURNED>
__global__ void __launch_bounds__(kThreads, 5)
    paged_append_rows_kernel(PagedArgs p, const IO* __restrict__ qkv, const int32_t* __restrict__ offsets, int rows,
                             IO* __restrict__ query_out, int parts, int part_heads) {
  griddep_wait();
  griddep_launch_dependents();
  append_rows<IO, CT, D, EXACT, TURNED>(p, qkv, offsets, rows, query_out, parts, part_heads, true,
                                        static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5));
}

// Chunks into a pool with bounds: the first blocks take the touched pages'
// keys, the others the rows' queries and values.
template <typename IO, typename CT, int D, bool EXACT, int kBlocks, bool TURNED>
__global__ void __launch_bounds__(kPageThreads, kBlocks)
    paged_append_chunks_kernel(PagedArgs p, const IO* __restrict__ qkv, const int32_t* __restrict__ offsets, int rows,
                               IO* __restrict__ query_out, int parts, int part_heads, int page_blocks, int page_heads) {
  griddep_wait();
  griddep_launch_dependents();
  if (static_cast<int>(blockIdx.x) < page_blocks)
    append_page<IO, CT, D, EXACT, TURNED>(p, qkv, offsets, rows, page_heads, blockIdx.x);
  else
    append_rows<IO, CT, D, EXACT, TURNED>(
        p, qkv, offsets, rows, query_out, parts, part_heads, false,
        static_cast<int64_t>(blockIdx.x - page_blocks) * (kPageThreads / 32) + (threadIdx.x >> 5));
}

// Bounds of the pages that a chunk touched, any shape: the block of a page's
// first new row walks the page's new slots.
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
    CT* at = static_cast<CT*>(p.bounds) + bounds_row(p, page, h, D) + d;
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

// The layers that append_rows takes.
bool by_rows(const tla_paged* P) {
  return P->wide && P->base.rotary % 8 == 0;
}
// Shared memory of the block-per-row kernel: the row in float32, its cosines and sines.
size_t row_smem(const tla_paged* P) {
  return sizeof(float) * (static_cast<size_t>(P->base.Hq + 2 * P->base.Hk) * P->base.D + P->base.rotary);
}

template <typename IO, typename CT, bool TURNED>
cudaError_t append_by_rows(const tla_paged* P, const PagedArgs& p, const void* qkv, const int32_t* offsets, int rows,
                           void* query_out, cudaStream_t stream) {
  const int D = p.a.D;
  const bool by_pages = p.bounds && offsets;
  // Warps per row: enough for 16 on every SM, at most one per warp-wide load
  // (64 rows of 48 heads: 12 warps per row).
  const int heads = p.a.Hq + (by_pages ? 1 : 2) * p.a.Hk, per = 256 / (D == 64 ? 64 : D <= 128 ? 128 : 256);
  const int most = (heads + per - 1) / per;
  long long parts = (16LL * P->base.ctx->sm_count + rows - 1) / rows;
  parts = parts < 1 ? 1 : parts > most ? most : parts;
  const int part_heads = (most + static_cast<int>(parts) - 1) / static_cast<int>(parts) * per;
  parts = (heads + part_heads - 1) / part_heads;
  if (!by_pages) {
    auto k = D == 64    ? paged_append_rows_kernel<IO, CT, 64, true, TURNED>
             : D == 128 ? paged_append_rows_kernel<IO, CT, 128, true, TURNED>
             : D < 128  ? paged_append_rows_kernel<IO, CT, 128, false, TURNED>
                        : paged_append_rows_kernel<IO, CT, 256, false, TURNED>;
    return launch_pdl(k, static_cast<unsigned>((rows * parts + 3) / 4), kThreads, 0, stream, p,
                      static_cast<const IO*>(qkv), offsets, rows, static_cast<IO*>(query_out),
                      static_cast<int>(parts), part_heads);
  }
  // a chunk of n rows touches at most (n - 1) / page_size + 2 pages, and no more than its rows
  const long long pages =
      min(static_cast<long long>(rows), (static_cast<long long>(rows) >> p.page_shift) + 2LL * p.batch);
  // kv heads per page block: all eight warps on one while that gives no more
  // than two blocks per SM (one or four: 24 and 23 us for 16 chunks of up to
  // 500 rows, 48 heads of 64, against 20)
  int page_heads = 1;
  while (page_heads < 8 && page_heads < p.a.Hk &&
         pages * ((p.a.Hk + page_heads - 1) / page_heads) > 2 * P->base.ctx->sm_count)
    page_heads *= 2;
  const long long blocks = pages * ((p.a.Hk + page_heads - 1) / page_heads);
  // Many blocks run four on an SM (64 registers each thread): more reads in
  // flight; few run three (84). Measured (three / four, us; * what the rule
  // takes), 32 + 8 + 8 heads of 128: 1 chunk of 2048 rows 17.1* / 15.2, of 8192
  // 41.8 / 37.6*, 16 of up to 256 16.5* / 17.2, of up to 1024 41.2 / 43.0*, of
  // up to 2047 95 / 88* (with QK-norm, token-major bfloat16 pages 104 / 93*);
  // the same heads of 64: 1 of 2048 10.2* / 8.9, 16 of up to 256 8.9* / 9.5, of
  // up to 2047 56 / 50*; 14 + 2 + 2 heads of 64: 1 of 2048 7.3* / 8.4. Widths
  // between and above have the three only.
  const int warps = kPageThreads / 32;
  const long long grid = blocks + (rows * parts + warps - 1) / warps;
  const bool many = grid > 6LL * P->base.ctx->sm_count;
  auto k = D < 128 ? paged_append_chunks_kernel<IO, CT, 128, false, 3, TURNED>
                   : paged_append_chunks_kernel<IO, CT, 256, false, 3, TURNED>;
  if (D == 64)
    k = many ? paged_append_chunks_kernel<IO, CT, 64, true, 4, TURNED>
             : paged_append_chunks_kernel<IO, CT, 64, true, 3, TURNED>;
  if (D == 128)
    k = many ? paged_append_chunks_kernel<IO, CT, 128, true, 4, TURNED>
             : paged_append_chunks_kernel<IO, CT, 128, true, 3, TURNED>;
  return launch_pdl(k, static_cast<unsigned>(grid), kPageThreads, 0, stream, p, static_cast<const IO*>(qkv), offsets,
                    rows, static_cast<IO*>(query_out), static_cast<int>(parts), part_heads, static_cast<int>(blocks),
                    page_heads);
}

template <typename IO, typename CT>
cudaError_t append_t(const tla_paged* P, const PagedArgs& p, const void* qkv, const int32_t* offsets, int rows,
                     void* query_out, cudaStream_t stream) {
  if (by_rows(P))
    return p.a.rotary == p.a.D && p.a.pair_count >= p.a.rotary / 2
               ? append_by_rows<IO, CT, true>(P, p, qkv, offsets, rows, query_out, stream)
               : append_by_rows<IO, CT, false>(P, p, qkv, offsets, rows, query_out, stream);
  const size_t smem = row_smem(P);
  auto k = paged_append_kernel<IO, CT>;
  cudaError_t e = cudaSuccess;
  if (smem > 48 * 1024) e = raise_smem_limit(reinterpret_cast<const void*>(k), static_cast<int>(smem));
  if (e != cudaSuccess) return e;
  e = launch_pdl(k, rows, kThreads, smem, stream, p, static_cast<const IO*>(qkv), offsets, rows,
                 static_cast<IO*>(query_out));
  if (e != cudaSuccess || !p.bounds || !offsets) return e;
  return launch_pdl(paged_bounds_kernel<CT>, rows, kThreads, 0, stream, p, offsets, rows);
}

}  // namespace

bool paged_append_takes(const tla_paged* P) { return by_rows(P) || row_smem(P) <= 227 * 1024; }

cudaError_t launch_paged_append(const tla_paged* P, const PagedArgs& p, const void* qkv, const int32_t* offsets,
                                int rows, void* query_out, cudaStream_t stream) {
  if (P->io == kFp16) return append_t<__half, __half>(P, p, qkv, offsets, rows, query_out, stream);
  if (P->io == kBf16) return append_t<__nv_bfloat16, __nv_bfloat16>(P, p, qkv, offsets, rows, query_out, stream);
  if (P->kept == kFp16) return append_t<float, __half>(P, p, qkv, offsets, rows, query_out, stream);
  if (P->kept == kBf16) return append_t<float, __nv_bfloat16>(P, p, qkv, offsets, rows, query_out, stream);
  return append_t<float, float>(P, p, qkv, offsets, rows, query_out, stream);
}

}  // namespace tla
