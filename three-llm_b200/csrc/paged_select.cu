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
#include <cooperative_groups.h>
#include <math.h>

#include <type_traits>

#include "paged.cuh"

namespace tla {

namespace cg = cooperative_groups;

namespace {

constexpr int kMaxWarps = 16;
constexpr int kMaxCluster = 8;
constexpr int kMaxHeld = 48 * 1024;  // ranks that one block's shared memory holds
constexpr int kScorePages = 32 * kMaxWarps;  // pages per block of the scoring kernel for longer sequences
// What a block gets without asking, its own variables counted in: 48 KB (and 1
// KB left over here for their padding).
constexpr size_t kDefaultSmem = 47 * 1024;

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

constexpr uint32_t kAlways = 0xffffffffu;  // the rank of a page that always takes part

// 16-bit values become doubles by placing their bits: exponent and mantissa in
// the high word, without a new bias, give the value times kScale, exactly, for
// subnormals too (the conversion instructions, one of them per element at an
// eighth of the rate, would bound the kernel). The vector carries 2^880 in
// return: no product over- or underflows, and a sum times kBack is the score.
// (A bound that is not finite counts as a large one.)
template <typename CT>
struct Bits;
template <>
struct Bits<__half> {
  static constexpr int kShift = 10;  // 5 + 10 bits, scaled by 2^-1008
  static constexpr double kForth = 0x1p880, kBack = 0x1p128;
};
template <>
struct Bits<__nv_bfloat16> {
  static constexpr int kShift = 13;  // 8 + 7 bits, scaled by 2^-896
  static constexpr double kForth = 0x1p880, kBack = 0x1p16;
};
template <>
struct Bits<float> {
  static constexpr double kForth = 1, kBack = 1;  // (converted)
};

// The score's vector (N, then P, as the bounds' order), formed by a block. With
// `lanes` lanes of `vec` neighbouring elements each, element d lies where a
// warp's 16-byte reads of its lanes' pairs (2 k, 2 k + 1) are neighbours.
__device__ __forceinline__ int vec_place(int d, int vec, int lanes) {
  const int lane = d / vec % lanes, e = d / (vec * lanes) * vec + d % vec;  // e: the lane's element
  return (e / 2 * lanes + lane) * 2 + (e & 1);
}
template <int kThreads, typename IO>
__device__ __forceinline__ void form_vector(const PagedArgs& p, const IO* query, int b, int kvh, double* vec, int per,
                                            int lanes, double scale) {
  const int D = p.a.D, G = p.a.G;
  const IO* q = query + (static_cast<int64_t>(b) * p.a.Hq + kvh * G) * D;
  for (int d = threadIdx.x; d < D; d += kThreads) {
    double neg = 0, pos = 0;
#pragma unroll 4
    for (int g = 0; g < G; ++g) {
      const float x = to_f32(q[g * D + d]);
      neg += fminf(x, 0.f);
      pos += fmaxf(x, 0.f);
    }
    vec[lanes ? vec_place(d, per, lanes) : d] = neg * scale;
    vec[lanes ? vec_place(D + d, per, lanes) : D + d] = pos * scale;
  }
}

// 16 bytes of bounds times their part of the vector.
template <typename CT>
__device__ __forceinline__ double dot16(uint4 u, const double* v) {
  double s0 = 0, s1 = 0;
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  if constexpr (sizeof(CT) == 2) {
    constexpr uint32_t kRest = 0x7fffu << Bits<CT>::kShift;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t even = (w[e] << 16 & 0x80000000u) | (w[e] << Bits<CT>::kShift & kRest);
      const uint32_t odd = (w[e] & 0x80000000u) | (w[e] >> (16 - Bits<CT>::kShift) & kRest);
      s0 = fma(v[2 * e], __hiloint2double(static_cast<int>(even), 0), s0);
      s1 = fma(v[2 * e + 1], __hiloint2double(static_cast<int>(odd), 0), s1);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
      s0 = fma(v[e], static_cast<double>(__uint_as_float(w[e])), s0);
      s1 = fma(v[e + 1], static_cast<double>(__uint_as_float(w[e + 1])), s1);
    }
  }
  return s0 + s1;
}

// A lane's page of a warp that takes pages first, first + step, ... of a
// sequence: the lane-th of them. Their table entries may be looked up before
// the range is known (`index` below the table's width).
__device__ __forceinline__ int raw_page(const PagedArgs& p, int b, int64_t index) {
  return index < p.width ? p.table[static_cast<int64_t>(b) * p.width + index] : -1;
}

// Ranks of 32 pages of a pair (i = from + step * lane, raw: their table
// entries), handed to `put(i, rank)` by their lanes. Each page's bounds are
// read across the lanes, kAhead reads in flight; kD is head_dim, or 0 for any.
template <typename CT, int kD, typename Put>
__device__ __forceinline__ void score_32(const PagedArgs& p, const double* vec, int kvh, PageRange r, int first,
                                         int last, int from, int step, int raw, const Put& put) {
  const unsigned full = 0xffffffffu;
  const int D = p.a.D, lane = threadIdx.x & 31;
  const int mine = from + step * lane;
  const bool held = mine < r.n, always = held && (mine < first || mine >= r.n - last);
  int page = held && !always ? raw : -1;
  if (page < -1 || page >= p.page_count || (page == -1 && held && !always)) {
    report_error(p.a.error, TLA_ERR_PAGE);
    page = -1;
  }
  if (held && page < 0) put(mine, always ? kAlways : 0u);  // (a page outside the pool ranks last)
  const unsigned scored = __ballot_sync(full, page >= 0);
  const CT* bounds = static_cast<const CT*>(p.bounds) + static_cast<int64_t>(kvh) * 2 * D;
  const int64_t stride = static_cast<int64_t>(p.a.Hk) * 2 * D;
  if constexpr (kD > 0) {
    constexpr int kVec = 16 / sizeof(CT), kReads = 2 * kD / kVec;        // 16-byte reads per page
    constexpr int kLanes = kReads < 32 ? kReads : 32, kPer = kReads / kLanes;  // lanes per page, reads per lane
    constexpr int kPages = 32 / kLanes, kMost = 8 / kPer;  // pages per warp-wide read; reads in flight
    const int sub = lane / kLanes, at = lane % kLanes;
    double v[kPer][kVec];
#pragma unroll
    for (int i = 0; i < kPer; ++i)
#pragma unroll
      for (int e = 0; e < kVec; e += 2) {
        const double2 x = reinterpret_cast<const double2*>(vec)[(i * kVec + e) / 2 * kLanes + at];
        v[i][e] = x.x;
        v[i][e + 1] = x.y;
      }
    const int n = 32 - __clz(scored);  // (0 when none is scored)
    auto round = [&](auto ahead, int k0) {
      constexpr int kAhead = decltype(ahead)::value;
      uint4 u[kAhead][kPer];
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        const int k = k0 + a * kPages + sub, of = __shfl_sync(full, page, k & 31);
#pragma unroll
        for (int i = 0; i < kPer; ++i)
          u[a][i] = of < 0 || k > 31
                        ? make_uint4(0, 0, 0, 0)
                        : *reinterpret_cast<const uint4*>(bounds + of * stride + (i * kLanes + at) * kVec);
      }
      double s[kAhead];
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        s[a] = dot16<CT>(u[a][0], v[0]);
#pragma unroll
        for (int i = 1; i < kPer; ++i) s[a] += dot16<CT>(u[a][i], v[i]);
      }
      // Sums across the page's lanes: as long as there are several pages, a
      // lane hands half of them over and goes on with the other half.
      int o = kLanes / 2;
#pragma unroll
      for (int left = kAhead; left > 1; left /= 2, o /= 2) {
#pragma unroll
        for (int a = 0; a < left / 2; ++a) {
          const bool upper = (lane & o) != 0;
          const double given = upper ? s[a] : s[a + left / 2];
          s[a] = (upper ? s[a + left / 2] : s[a]) + __shfl_xor_sync(full, given, o);
        }
      }
      constexpr int kOwners = kLanes / kAhead;  // lanes that end up with the same page
#pragma unroll
      for (int o2 = kOwners / 2; o2 > 0; o2 /= 2) s[0] += __shfl_xor_sync(full, s[0], o2);
      const int k = k0 + at / kOwners * kPages + sub;
      if (at % kOwners == 0 && (scored >> (k & 31) & 1) && k < 32)
        put(from + step * k, min(rank_of(static_cast<float>(s[0] * Bits<CT>::kBack)), 0xfffffffeu));
    };
    int k0 = 0;
    for (; n - k0 > 2 * kPages; k0 += kMost * kPages) round(std::integral_constant<int, kMost>(), k0);
    for (; k0 < n; k0 += kPages) round(std::integral_constant<int, 1>(), k0);
  } else {
    for (unsigned left = scored; left != 0; left &= left - 1) {
      const int k = __ffs(left) - 1, of = __shfl_sync(full, page, k);
      double s = 0;
      for (int d = lane; d < 2 * D; d += 32) s = fma(vec[d], static_cast<double>(to_f32(bounds[of * stride + d])), s);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(full, s, o);
      if (lane == k) put(mine, min(rank_of(static_cast<float>(s)), 0xfffffffeu));
    }
  }
}
// Lanes that hold a page's 16-byte pieces (0: any other head_dim).
template <typename CT>
__device__ __forceinline__ int piece_lanes(int D) {
  const int reads = 2 * D * static_cast<int>(sizeof(CT)) / 16;
  return D == 64 || D == 128 || D == 256 ? min(reads, 32) : 0;
}
template <typename CT, typename Put>
__device__ __forceinline__ void score_any(const PagedArgs& p, const double* vec, int kvh, PageRange r, int first,
                                          int last, int from, int step, int raw, const Put& put) {
  if (p.a.D == 128)
    score_32<CT, 128>(p, vec, kvh, r, first, last, from, step, raw, put);
  else if (p.a.D == 64)
    score_32<CT, 64>(p, vec, kvh, r, first, last, from, step, raw, put);
  else if (p.a.D == 256)
    score_32<CT, 256>(p, vec, kvh, r, first, last, from, step, raw, put);
  else
    score_32<CT, 0>(p, vec, kvh, r, first, last, from, step, raw, put);
}

// Writes the `count` pages of the highest ranks, ties to the lower page, in
// page order, by one block. The lowest rank that is taken is found below the
// leading bits that the lowest and highest rank share, 9 to 11 bits at a time
// (four table entries per thread): a table of counts (like pages' ranks agree in their leading bits, so the bits
// below spread them over the table), then a scan from its top; it ends early
// when every rank of the border's entry is taken. The list is written in one
// pass in which a thread owns four neighbouring pages. What this costs is
// barriers: seven or eight in all for 2048 pages, 1.7 us.
struct PickSmem {
  uint32_t low[kMaxWarps], high[kMaxWarps];
  int sums[2][kMaxWarps];
  int digit, want, here;
  __align__(16) int bins[4 * kMaxWarps * 32];
};

// Sums of the lanes up to and with this one.
__device__ __forceinline__ int warp_scan(int v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int n = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += n;
  }
  return v;
}

template <int kThreads>
__device__ __forceinline__ void pick_pages(const uint32_t* rank, PageRange r, int count, int always, int32_t* out,
                                           PickSmem* sm) {
  constexpr int kWarps = kThreads / 32, kOwn = 4, kPickBins = kOwn * kThreads;
  constexpr int kPickBits = kThreads == 512 ? 11 : kThreads == 256 ? 10 : 9;
  static_assert(1 << kPickBits == kPickBins, "a table entry per value of the bits");
  const unsigned full = 0xffffffffu;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int want = count - always;  // of the ranks below kAlways that agree with the prefix
  uint32_t prefix = 0;
  int shift = 32;  // the prefix's bits from here up are found
  if (want > 0) {
    uint32_t low = 0xffffffffu, high = 0u;
    for (int i = tid; i < r.n; i += kThreads) {
      const uint32_t v = rank[i];
      low = min(low, v);
      high = max(high, v == kAlways ? 0u : v);
    }
    low = __reduce_min_sync(full, low);
    high = __reduce_max_sync(full, high);
    if (lane == 0) {
      sm->low[warp] = low;
      sm->high[warp] = high;
    }
    __syncthreads();
    low = __reduce_min_sync(full, lane < kWarps ? sm->low[lane] : 0xffffffffu);
    high = __reduce_max_sync(full, lane < kWarps ? sm->high[lane] : 0u);
    // (n > count, so there is a rank below kAlways, and low <= high)
    shift = low == high ? 0 : 32 - __clz(low ^ high);
    prefix = shift >= 32 ? 0u : high >> shift << shift;
    while (shift > 0) {
      const int bits = min(kPickBits, shift), next = shift - bits;
      for (int i = tid; i < kPickBins / 4; i += kThreads) reinterpret_cast<int4*>(sm->bins)[i] = make_int4(0, 0, 0, 0);
      __syncthreads();
      for (int i = tid; i < r.n; i += kThreads) {
        const uint32_t v = rank[i];
        if (v != kAlways && (shift >= 32 || (v ^ prefix) >> shift == 0))
          atomicAdd(&sm->bins[(v >> next) & ((1 << bits) - 1)], 1);
      }
      __syncthreads();
      // thread t owns the t-th kOwn entries from the top
      const int top = kPickBins - 1 - tid * kOwn;
      int own = 0;
#pragma unroll
      for (int k = 0; k < kOwn; ++k) own += sm->bins[top - k];
      const int scan = warp_scan(own, lane);
      if (lane == 31) sm->sums[0][warp] = scan;
      __syncthreads();
      int above = scan - own + __reduce_add_sync(full, lane < warp ? sm->sums[0][lane] : 0);
      if (above < want && above + own >= want) {
        int k = 0;
        while (above + sm->bins[top - k] < want) above += sm->bins[top - k++];
        sm->digit = top - k;
        sm->want = want - above;
        sm->here = sm->bins[top - k];
      }
      __syncthreads();
      prefix |= static_cast<uint32_t>(sm->digit) << next;
      want = sm->want;
      shift = next;
      if (sm->here == want) break;
    }
  }
  // taken: kAlways, ranks above the prefix from `shift` up, and the first `want` that agree with it
  const uint32_t border = shift >= 32 ? 0u : prefix >> shift;
  int taken = 0, equal = 0;  // in the rounds before; a round's counts share a word
  bool buffer = false;
  for (int base = 0; base < r.n; base += 4 * kThreads) {
    const int i0 = base + 4 * tid;
    int surely = 0, same = 0;  // one bit per page
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t v = i0 + e < r.n ? rank[i0 + e] : 0u;
      const bool sure = v == kAlways || (shift < 32 && v >> shift > border);
      if (i0 + e < r.n) {
        surely |= sure << e;
        same |= (!sure && shift < 32 && v >> shift == border) << e;
      }
    }
    const int own = __popc(surely) << 16 | __popc(same), scan = warp_scan(own, lane);
    if (lane == 31) sm->sums[buffer][warp] = scan;
    __syncthreads();
    const int s = lane < kWarps ? sm->sums[buffer][lane] : 0;
    const int all = __reduce_add_sync(full, s), prior = __reduce_add_sync(full, lane < warp ? s : 0) + scan - own;
    buffer = !buffer;
    int sure_n = taken + (prior >> 16), same_n = equal + (prior & 0xffff);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool is_sure = surely >> e & 1, is_same = same >> e & 1;
      if (is_sure || (is_same && same_n < want)) out[sure_n + min(same_n, want)] = r.begin + i0 + e;
      sure_n += is_sure;
      same_n += is_same;
    }
    taken += all >> 16;
    equal += all & 0xffff;
  }
}

// All of a pair's pages, when there are no more than `count`.
template <int kThreads>
__device__ __forceinline__ void list_all(const PagedArgs& p, int pos, PageRange r, int count, int32_t* out) {
  if (r.n == 0 && pos >= 0 && threadIdx.x == 0) report_error(p.a.error, TLA_ERR_POSITION);
  for (int i = threadIdx.x; i < count; i += kThreads) out[i] = i < r.n ? r.begin + i : -1;
}

// A cluster per (sequence, kv head): its warps score every so many-th page
// each and leave the ranks in the first block's shared memory, which picks.
// One launch: what a step waits for here is latency, not the bounds' bytes, so
// the position, the query and the first table entries are read side by side.
template <typename IO, typename CT, int kThreads>
__global__ void __launch_bounds__(kThreads, kThreads == 512 ? 1 : kThreads == 256 ? 2 : 5)
    paged_select_kernel(PagedArgs p, const IO* __restrict__ query, int first, int last, int count,
                        int32_t* __restrict__ pages_out) {
  extern __shared__ __align__(16) double vec[];  // [2][D], then the ranks
  __shared__ PickSmem pick_s;
  constexpr int kWarps = kThreads / 32;
  uint32_t* ranks = reinterpret_cast<uint32_t*>(vec + 2 * p.a.D);
  griddep_wait();
  griddep_launch_dependents();
  cg::cluster_group cluster = cg::this_cluster();
  const int share = cluster.block_rank(), shares = cluster.num_blocks();
  if (shares > 1) cluster.barrier_arrive();
  const int pair = blockIdx.x / shares, b = pair / p.a.Hk, kvh = pair - b * p.a.Hk;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int step = kWarps * shares;
  int from = warp * shares + share;
  const int pos = p.positions[b];
  int raw = p.a.sliding == 0 ? raw_page(p, b, from + static_cast<int64_t>(step) * lane) : 0;
  form_vector<kThreads>(p, query, b, kvh, vec, 16 / static_cast<int>(sizeof(CT)), piece_lanes<CT>(p.a.D),
              piece_lanes<CT>(p.a.D) ? Bits<CT>::kForth : 1);
  const PageRange r = page_range(p, pos);
  int32_t* out = pages_out + static_cast<int64_t>(pair) * count;
  // every block of the cluster runs before one writes into another's memory
  if (shares > 1) cluster.barrier_wait();
  if (r.n <= count) {  // (the same for the whole cluster)
    if (share == 0) list_all<kThreads>(p, pos, r, count, out);
    return;
  }
  __syncthreads();
  uint32_t* held = shares > 1 ? cluster.map_shared_rank(ranks, 0) : ranks;
  for (bool again = false; from < r.n; from += 32 * step, again = true) {
    if (again || p.a.sliding > 0) raw = raw_page(p, b, r.begin + from + static_cast<int64_t>(step) * lane);
    score_any<CT>(p, vec, kvh, r, first, last, from, step, raw, [&](int i, uint32_t rank) { held[i] = rank; });
  }
  if (shares > 1)
    cluster.sync();
  else
    __syncthreads();
  if (share == 0) pick_pages<kThreads>(ranks, r, count, first + last, out, &pick_s);
}

// The same in two launches, the ranks in the workspace, for sequences of more
// pages than shared memory holds ranks.
template <typename IO, typename CT>
__global__ void __launch_bounds__(kMaxWarps * 32)
    paged_score_kernel(PagedArgs p, const IO* __restrict__ query, int first, int last, int count,
                       uint32_t* __restrict__ ranks) {
  extern __shared__ __align__(16) double vec[];
  griddep_wait();
  griddep_launch_dependents();
  const int kvh = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int b = blockIdx.z; b < p.batch; b += gridDim.z) {
    const PageRange r = page_range(p, p.positions[b]);
    const int from = blockIdx.x * kScorePages + warp * 32;
    if (r.n <= count || blockIdx.x * kScorePages >= r.n) continue;
    __syncthreads();
    form_vector<kMaxWarps * 32>(p, query, b, kvh, vec, 16 / static_cast<int>(sizeof(CT)), piece_lanes<CT>(p.a.D),
              piece_lanes<CT>(p.a.D) ? Bits<CT>::kForth : 1);
    __syncthreads();
    uint32_t* held = ranks + (static_cast<int64_t>(b) * p.a.Hk + kvh) * p.width;
    if (from < r.n)
      score_any<CT>(p, vec, kvh, r, first, last, from, 1, raw_page(p, b, r.begin + from + static_cast<int64_t>(lane)),
                    [&](int i, uint32_t rank) { held[i] = rank; });
  }
}
__global__ void __launch_bounds__(kMaxWarps * 32)
    paged_pick_kernel(PagedArgs p, const uint32_t* __restrict__ ranks, int always, int count,
                      int32_t* __restrict__ pages_out) {
  __shared__ PickSmem pick_s;
  griddep_wait();
  griddep_launch_dependents();
  const int pos = p.positions[blockIdx.x / p.a.Hk];
  const PageRange r = page_range(p, pos);
  int32_t* out = pages_out + static_cast<int64_t>(blockIdx.x) * count;
  if (r.n <= count)
    list_all<kMaxWarps * 32>(p, pos, r, count, out);
  else
    pick_pages<kMaxWarps * 32>(ranks + static_cast<int64_t>(blockIdx.x) * p.width, r, count, always, out, &pick_s);
}

// Pages that a sequence can have in this call.
int most_pages(int width, int shift, int capacity) {
  const long long n = (static_cast<long long>(capacity) + (1 << shift) - 1) >> shift;
  return static_cast<int>(n < width ? n : width);
}

template <typename IO, typename CT>
cudaError_t select_t(const tla_paged* P, const PagedArgs& p, const void* query, int first, int last,
                     int32_t* pages_out, int count, uint32_t* ranks, cudaStream_t stream) {
  const int most = most_pages(p.width, p.page_shift, p.capacity);
  const long long pairs = static_cast<long long>(p.batch) * p.a.Hk;
  const size_t vec = 2 * p.a.D * sizeof(double);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.blockDim = dim3(kMaxWarps * 32);
  if (most <= kMaxHeld) {
    // Larger blocks for longer sequences, whose first one picks alone, its rounds
    // and the list's writing going over all pages; small ones, of which an SM
    // runs more threads, where the pairs alone give every SM something to do
    // while another picks. A cluster's blocks share the scores out, up to eight,
    // at least two pages per warp, as long as all blocks run at once (five per
    // SM of 128 threads, two of 256, one of 512; the longest ones up to 1.6
    // times that). Measured (threads x blocks per pair, us; * what the rule
    // takes): 512 pairs of 64 pages 128 x 1 7.3*, x 2 13.0; 160 of 1250 (128
    // wide) 128 x 4 36.7*, 256 x 1 53, 512 x 2 52; 256 of 256 (128 wide) 128 x 1
    // 20.6, x 2 16.6*, x 4 19.1, 256 x 1 14.6, of ragged lengths up to that 128 x
    // 1 14.5, x 2 12.5*, x 4 11.8, 256 x 1 12.0; 256 of 4000 256 x 1 91*, 128 x 2
    // 109, 512 x 2 111; 128 of 256 (128 wide) 128 x 4 10.1*, 256 x 2 8.9; 64 of
    // 500 (128 wide) 256 x 4 9.3*, x 8 15.2; 32 of 1024 (128 wide) 256 x 8 13.5*,
    // x 4 11.5, 512 x 2 12.8; 114 of up to 5562 512 x 2 46*, x 8 60; 32 of 1875
    // 512 x 4 13.8*, x 8 22.2; 8 of 2048 (128 wide) 512 x 8 9.9*, x 2 20.
    // (Clusters of 16 leave a GPC's other SMs idle: 8 of them with 512 threads
    // each ran in two waves, 28 us for a sparse step at 131072 tokens.)
    const int sms = P->base.ctx->sm_count;
    auto k = paged_select_kernel<IO, CT, 128>;
    int warps = 4, blocks = 5 * sms;
    if (most > (pairs <= sms ? 256 : 1536)) k = paged_select_kernel<IO, CT, 256>, warps = 8, blocks = 2 * sms;
    if (most > 1024 && pairs <= sms) k = paged_select_kernel<IO, CT, 512>, warps = 16, blocks = sms * 8 / 5;
    int shares = 1;
    while (shares < kMaxCluster && pairs * shares * 2 <= blocks && most > 2 * warps * shares) shares *= 2;
    const size_t smem = vec + (most > count ? most * sizeof(uint32_t) : 0);
    if (smem + sizeof(PickSmem) > kDefaultSmem) {
      const cudaError_t e = raise_smem_limit(reinterpret_cast<const void*>(k), static_cast<int>(smem));
      if (e != cudaSuccess) return e;
    }
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = shares;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(pairs * shares));
    cfg.blockDim = dim3(warps * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, k, p, static_cast<const IO*>(query), first, last, count, pages_out);
  }
  cfg.gridDim = dim3((most + kScorePages - 1) / kScorePages, p.a.Hk, p.batch < 65535 ? p.batch : 65535);
  cfg.dynamicSmemBytes = vec;
  const cudaError_t e =
      cudaLaunchKernelEx(&cfg, paged_score_kernel<IO, CT>, p, static_cast<const IO*>(query), first, last, count, ranks);
  if (e != cudaSuccess) return e;
  return launch_pdl(paged_pick_kernel, static_cast<unsigned>(pairs), kMaxWarps * 32, 0, stream, p,
                    static_cast<const uint32_t*>(ranks), first + last, count, pages_out);
}

}  // namespace

size_t paged_select_workspace(const tla_paged* P, int batch, int width) {
  const PagedArgs p = paged_args(P, nullptr, nullptr, width, batch);
  if (!P->pool.bounds || most_pages(width, P->page_shift, p.capacity) <= kMaxHeld) return 0;
  return static_cast<size_t>(batch) * P->base.Hk * width * sizeof(uint32_t);
}

cudaError_t launch_paged_select(const tla_paged* P, const PagedArgs& p, const void* query, int first, int last,
                                int32_t* pages_out, int count, void* workspace, cudaStream_t stream) {
  uint32_t* ranks = static_cast<uint32_t*>(workspace);
  if (P->io == kFp16) return select_t<__half, __half>(P, p, query, first, last, pages_out, count, ranks, stream);
  if (P->io == kBf16)
    return select_t<__nv_bfloat16, __nv_bfloat16>(P, p, query, first, last, pages_out, count, ranks, stream);
  if (P->kept == kFp16) return select_t<float, __half>(P, p, query, first, last, pages_out, count, ranks, stream);
  if (P->kept == kBf16) return select_t<float, __nv_bfloat16>(P, p, query, first, last, pages_out, count, ranks, stream);
  return select_t<float, float>(P, p, query, first, last, pages_out, count, ranks, stream);
}

}  // namespace tla
