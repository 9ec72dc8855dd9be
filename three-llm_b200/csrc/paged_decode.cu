// Split-KV decode over a paged cache (sm_100a): 16-bit pages of 16 tokens and
// up, head_dim a multiple of 8 up to 256 (the kernel is built for 64, 128 and
// 256, whose columns past head_dim stay zero in shared memory).
//
//   o = sum_t 2^(x_t - m) v_t / sum_t 2^(x_t - m),  x_t = log2(e) scale q.k_t
//
// Each K and V element is read once and used by the group's query heads, about
// 2 G operations per byte: memory bounds it, so the kernel's shape follows the
// reads. A (sequence, kv head) pair's tokens are cut into tiles (32 tokens at
// head_dim 64, 16 above: 8 KB of K and V at 64 and 128), and the tiles of all pairs into
// equal contiguous shares, one per resident CTA, whatever the sequences'
// lengths; a share may begin and end inside a pair. Four warps take a share's
// tiles in turn, each by itself: a warp keeps a ring of tiles of its own, which
// its lanes fill by asynchronous 16-byte copies (any order, padding and stride
// of pages, heads and slots), so that no barrier, no producer and no other
// warp's tile stands between its reads. Its page table entries are looked up
// 32 at a time, one window ahead, and its copies run ahead of its products
// across the ends of sequences. 16 tokens always lie in one page: a page's end
// inside a tile, a page that is not in the pool and the window's edges are
// decided when a row is copied, as zeros in place of it.
//
// (A version with a producer warp and one TMA box per page piece moved the
// same bytes per second when every SM streams, but a tile took one CTA 0.43 us
// at 64-token pages and 0.7 us at 16: the issue of up to 8 boxes per tile and
// the round trip of a stage bound it.)
//
// S^T = K Q^T and O^T += V^T P^T run as m16n8k16 tensor-core tiles: the tokens
// (then the dimensions) are the 16 rows and the group's query heads the 8
// columns (two column tiles for groups over 8), so that groups of 8 and fewer
// waste no half of a tile, and P^T moves from accumulators to an operand by
// one 8 x 8 transposition per 8 tokens.
//
// Pairs that several CTAs share leave (m, l, o) triples in the caller's
// workspace, which a second kernel joins: no counters, so nothing has to be
// prepared or survives the call.
//
// Each softmax weight goes to the tensor cores in two parts of the pages' type,
// the weight cut off and what that left: 21 bits over float16 pages (down to
// 2^-18 of the largest weight, below that 2^-39 of it: see kLiftOf), 15 over
// bfloat16. The output's own rounding is then all that a 16-bit call rounds: its
// error against 64 bits is 2.1e-4 (float16) and 1.7e-3 (bfloat16), where weights
// in one part made 2.7e-4 and 2.2e-3 of it. The second products cost 1 to 2% (8
// x 4097 tokens 16.8 us for 16.5, 64 ragged 136.0 for 135.5), 5% with 16 query
// heads per kv head (8 x 4097 19.6 us for 18.7).
//
// float32 activations over float16 pages: each query row is scaled by a power
// of two and split the same way, so that the scores carry 21 bits as well, and
// the output keeps float32's use for its caller. K and V are exact as stored.
#include <cooperative_groups.h>
#include <math.h>

#include <type_traits>

#include "paged.cuh"

namespace tla {

namespace cg = cooperative_groups;

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kMaxBatch = 1024;  // prefix table in shared memory
constexpr int kCtasPerSm = 2;
constexpr int kMaxCluster = 16;
constexpr int kMaxGrid = 1024;   // segment table of the joining kernel
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kNowhere = -(1 << 30);  // first position of 16 tokens that take no part

template <int D>
struct Cfg {
  static constexpr int kTile = D == 64 ? 32 : 16;
  static constexpr int kGroups = kTile / 16;
  static constexpr int kStages = 2;
  static constexpr int kTileBytes = kTile * D * 2;
  static constexpr int kStageBytes = 2 * kTileBytes;
  static constexpr int kQPitch = D * 2 + 16;
  // A pair costs its query set-up and its epilogue besides its tiles: counted
  // as this many tiles when the shares are cut.
  static constexpr int kSetup = 14;
};

// Byte offset of 16-byte piece `chunk` of token `tok` in a tile: the piece's
// place among its row's eighths turns with the token, so that the eight rows of
// a matrix operand lie in different banks.
template <int D>
__device__ __forceinline__ uint32_t tile_at(int tok, int chunk) {
  return static_cast<uint32_t>(tok * D * 2 + ((chunk ^ (tok & 7)) << 4));
}

struct DecodeParams {
  PagedArgs p;
  const void* query;
  const int32_t* pages;  // null, or [batch][Hk][count]
  const void* gate;
  void* out;
  float* scratch;  // [grid][2][rows][D + 2]
  long long scratch_floats;  // its extent (bounds-check builds)
  int count;
  int subs;        // groups of up to 16 query heads per kv head
  int rows;        // query heads per such group, the last one's may be fewer
  int small_grid;
  int cluster;     // CTAs per pair, joined within their cluster; 0: shares over all pairs
};

struct SmemLayout {
  int stages, q, red, part, meta, prefix, total;
};
template <int D>
__host__ __device__ inline SmemLayout smem_layout(int rows, int batch, bool split) {
  using C = Cfg<D>;
  SmemLayout s;
  int off = 0;
  s.stages = off;
  off += kWarps * C::kStages * C::kStageBytes;
  s.q = off;
  off += (split ? 2 : 1) * 16 * C::kQPitch;
  s.red = off;
  off += kWarps * rows * (D + 2) * 4;
  s.part = off;  // the CTA's triple for its cluster
  off += rows * (D + 2) * 4;
  off = (off + 15) & ~15;
  s.meta = off;
  off += kWarps * C::kStages * C::kGroups * 4;
  s.prefix = off;
  off += (2 * batch + 2) * 4;  // unit prefix, then positions
  s.total = off + 1024;  // alignment slack
  return s;
}

// What a sequence's pairs walk: tiles [first, first + n) of its tokens, or of
// its listed pages' tokens (then first is 0 and n counts the longest list).
struct Walk {
  int lo, hi, first, tiles;
};
template <int D>
__device__ __forceinline__ Walk walk_of(const DecodeParams& d, int pos) {
  constexpr int kTile = Cfg<D>::kTile;
  Walk w;
  if (!paged_range(d.p, pos, &w.lo, &w.hi)) return {0, -1, 0, 0};
  if (d.pages) {
    const long long n = min(d.count, (w.hi >> d.p.page_shift) + 1);
    w.first = 0;
    w.tiles = static_cast<int>(((n << d.p.page_shift) + kTile - 1) / kTile);
  } else {
    w.first = w.lo / kTile;
    w.tiles = w.hi / kTile - w.first + 1;
  }
  return w;
}

template <int D>
__device__ __forceinline__ int units_of(const DecodeParams& d, int pos) {
  const int tiles = walk_of<D>(d, pos).tiles;
  return tiles > 0 ? (tiles + Cfg<D>::kSetup) * d.p.a.Hk * d.subs : 0;
}

// Inclusive scan of prefix[1..batch] by one warp (prefix[0] = 0).
__device__ __forceinline__ void scan_prefix(int* prefix, int batch, int lane) {
  int carry = 0;
  for (int base = 1; base <= batch; base += 32) {
    const int i = base + lane;
    int v = i <= batch ? prefix[i] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int n = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += n;
    }
    if (i <= batch) prefix[i] = v + carry;
    carry += __shfl_sync(0xffffffffu, v, 31);
  }
}

// The CTAs that share a launch's units: few units go to one CTA per SM, so
// that fewer triples have to be joined.
__device__ __forceinline__ int effective_grid(int total, int grid, int small) {
  return small < grid && total < 8 * small ? small : grid;
}
// First unit of share c (a 64-bit division is on every CTA's way: only where 32 bits do not hold the product).
__device__ __forceinline__ int cta_begin(int c, int total, int grid) {
  if (total < (1 << 30) / kMaxGrid)
    return static_cast<int>(static_cast<unsigned>(c * total) / static_cast<unsigned>(grid));
  return static_cast<int>(static_cast<long long>(c) * total / grid);
}
// Largest c with cta_begin(c) <= g.
__device__ __forceinline__ int cta_of(int g, int total, int grid) {
  int c = total < (1 << 30) / kMaxGrid
              ? static_cast<int>(static_cast<unsigned>(g * grid) / static_cast<unsigned>(total))
              : static_cast<int>(static_cast<long long>(g) * grid / total);
  while (c + 1 < grid && cta_begin(c + 1, total, grid) <= g) ++c;
  while (c > 0 && cta_begin(c, total, grid) > g) --c;
  return c;
}

// The pair of sequence b that holds unit g, and the tiles [lt, lt + n) of it
// that a share ending at te takes from there.
struct Seg {
  int pair, tiles, lt, n;
  int start, next;  // the pair's first unit (its set-up units included), and where the share goes on
};
template <int D>
__device__ __forceinline__ Seg seg_at(const int* prefix, int b, int pairs, int g, int te) {
  Seg s;
  const int per = (prefix[b + 1] - prefix[b]) / pairs;
  s.tiles = per - Cfg<D>::kSetup;
  s.pair = (g - prefix[b]) / per;
  s.start = prefix[b] + s.pair * per;
  const int first = s.start + Cfg<D>::kSetup, end = min(te, s.start + per);
  s.lt = max(0, g - first);
  s.n = max(0, end - (first + s.lt));
  s.next = end;
  return s;
}

// 16 bytes to shared memory; zeros instead when `bytes` is 0.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy16_or_zeros(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <typename T>
__device__ __forceinline__ void mma_t(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  mma_16816(d, a, b0, b1);
}
template <>
__device__ __forceinline__ void mma_t<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  return pack_half2(lo, hi);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}
// The two values of a packed pair.
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
  return __half22float2(*reinterpret_cast<__half2*>(&v));
}
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) {  // a float's upper half
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
// A pair of values in two pairs of parts: the values cut off to T, and what that
// left, both of the values' sign. The parts are of the values times kUp, the next
// float after 1, so that the second is not zero either, and an infinity that a
// part is multiplied with stays one: two parts of different signs, or a zero,
// would make it a NaN.
constexpr float kUp = 1.f + 0x1p-23f;
template <typename T>
__device__ __forceinline__ uint32_t pack2_cut(float lo, float hi) {
  uint32_t v;
  if constexpr (std::is_same<T, __half>::value)
    asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(v) : "f"(hi), "f"(lo));
  else
    asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(v) : "f"(hi), "f"(lo));
  return v;
}
template <typename T>
__device__ __forceinline__ uint32_t pack2_rest(uint32_t cut, float lo, float hi) {
  const float2 f = unpack2<T>(cut);
  return pack2<T>(fmaf(lo, kUp, -f.x), fmaf(hi, kUp, -f.y));
}

// An 8 x 8 matrix of 16-bit values, a row pair of which each lane holds, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// 1 / sum, or 0 where no token took part.
__device__ __forceinline__ float inverse(float sum) { return sum != 0.f ? 1.f / sum : 0.f; }
// An output v (times inverse(sum)) and its gate; zero, whatever the gate holds,
// where no token took part.
template <typename IO>
__device__ __forceinline__ void store_out(const DecodeParams& d, int64_t i, float v, float inv) {
  v *= inv;
  if (d.gate && inv != 0.f) v = v * (1.f / (1.f + expf(-to_f32(static_cast<const IO*>(d.gate)[i]))));  // math.ts:271-273
  static_cast<IO*>(d.out)[i] = from_f32<IO>(v);
}

// Weights are formed as powers of two over a base that lies this far below the
// running maximum, the largest being 2^14: float16 keeps a weight's 11 bits down
// to 2^-28 of the largest, and rounds by 2^-39 of it at most below, where
// weights of up to 1 would be cut to ever fewer bits from 2^-14 on and vanish
// under 2^-25 (8192 of them together were lost or a third too heavy). The sum
// and the output carry the same factor. The base is rounded upwards, so that no
// weight passes 2^14 where scores are so large that a float's step is (there the
// base is the maximum itself). bfloat16 has float32's exponents.
template <typename CT>
constexpr float kLiftOf = std::is_same<CT, __half>::value ? 14.f : 0.f;

// SPLIT: float32 activations over float16 pages. TWO: more than 8 query heads per group.
template <int D, typename CT, bool SPLIT, bool TWO>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) paged_decode_kernel(const __grid_constant__ DecodeParams d) {
  using C = Cfg<D>;
  using IO = typename std::conditional<SPLIT, float, CT>::type;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const PagedArgs& p = d.p;
  const int Hq = p.a.Hq, G = p.a.G, pairs = p.a.Hk * d.subs, rows = d.rows, hd = p.a.D;
  const SmemLayout L = smem_layout<D>(rows, d.cluster ? 0 : p.batch, SPLIT);
  int* prefix = reinterpret_cast<int*>(smem + L.prefix);
  int* spos = prefix + p.batch + 1;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, cta = blockIdx.x;
  const uint32_t ring = smem_u32(smem + L.stages) + warp * C::kStages * C::kStageBytes;
  int* meta = reinterpret_cast<int*>(smem + L.meta) + warp * C::kStages * C::kGroups;  // first position of each 16 tokens
  if (tid == 0) prefix[0] = 0;
  if (hd < D)  // columns that no copy goes to
    for (int i = lane; i < C::kStages * C::kStageBytes / 16; i += 32)
      asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(ring + i * 16), "r"(0) : "memory");
  __syncwarp();
  griddep_wait();
  griddep_launch_dependents();
  int tb = 0, te = 1;  // the share's units; one segment with a cluster per pair
  Seg only;
  int only_b = 0, only_pos = 0;
  if (d.cluster) {
    const int all = cta / d.cluster, rank = cta - all * d.cluster;
    only_b = all / pairs;
    only_pos = p.positions[only_b];
    only.pair = all - only_b * pairs;
    if (only_pos >= p.capacity && tid == 0 && rank == 0) report_error(p.a.error, TLA_ERR_POSITION);
    only.tiles = walk_of<D>(d, only_pos).tiles;
    only.lt = rank * only.tiles / d.cluster;
    only.n = (rank + 1) * only.tiles / d.cluster - only.lt;
    only.start = 0;
    only.next = 1;
    if (only.tiles == 0) {  // (the same for the whole cluster) no sequence: zeros
      const int kvh = only.pair / d.subs, sub = only.pair - kvh * d.subs;
      const int h0 = kvh * G + sub * rows, heads = min(rows, (kvh + 1) * G - h0);
      for (int i = tid; rank == 0 && i < heads * hd; i += kThreads)
        static_cast<IO*>(d.out)[(static_cast<int64_t>(only_b) * Hq + h0) * hd + i] = from_f32<IO>(0.f);
      return;
    }
  } else {
    for (int b = tid; b < p.batch; b += kThreads) {
      const int pos = p.positions[b];
      if (pos >= p.capacity && cta == 0) report_error(p.a.error, TLA_ERR_POSITION);
      spos[b] = pos;
      prefix[b + 1] = units_of<D>(d, pos);
    }
    __syncthreads();
    if (warp == 0) scan_prefix(prefix, p.batch, lane);
    __syncthreads();
    const int total = prefix[p.batch];
    // rows without a sequence, spread over the whole launch
    for (int b = cta; b < p.batch; b += gridDim.x)
      if (prefix[b + 1] == prefix[b])
        for (int i = tid; i < Hq * hd; i += kThreads)
          static_cast<IO*>(d.out)[static_cast<int64_t>(b) * Hq * hd + i] = from_f32<IO>(0.f);
    const int grid = effective_grid(total, gridDim.x, d.small_grid);
    if (total == 0 || cta >= grid) return;
    tb = cta_begin(cta, total, grid);
    te = cta_begin(cta + 1, total, grid);
    if (tb >= te) return;
  }
  // the segment at unit g, *b its sequence (found from the one before)
  auto segment = [&](int* b, int g) -> Seg {
    if (d.cluster) {
      *b = only_b;
      return only;
    }
    while (prefix[*b + 1] <= g) ++*b;
    return seg_at<D>(prefix, *b, pairs, g, te);
  };
  auto walk = [&](int b) -> Walk { return walk_of<D>(d, d.cluster ? only_pos : spos[b]); };
  const int shift = p.page_shift, mask = (1 << shift) - 1;

  // ================================================================== copies
  // The warp's copies: tiles ld.it = warp, warp + 4, ... of the share, counted
  // over its segments, each into the ring's next stage.
  struct {
    int g, b, it, begin, end;          // the share's tiles [begin, end) are the current segment's
    int first, lo, hi, e_first, e_end;  // its first tile, range, and table (or list) entries
    int base, index, page, index_next, page_next;  // windows of 32 entries: a lane's page in the sequence and the pool
    const int32_t* list;
    int64_t head;  // the kv head's first element of a page
  } ld;
  ld.g = tb;
  ld.b = 0;
  ld.it = warp;
  ld.begin = ld.end = 0;
  ld.base = 0;
  ld.list = nullptr;
  // (Entries are only looked at when they are used, so that a window's loads
  // are not waited for; a list's end is checked there, too.)
  auto look = [&](int e, int* index, int* page) {
    const bool in = e >= ld.e_first && e < ld.e_end;
    *index = !in ? -1 : ld.list ? ld.list[e] : e;
    *page = static_cast<unsigned>(*index) < static_cast<unsigned>(p.width)
                ? p.table[static_cast<int64_t>(ld.b) * p.width + *index] : kNowhere;
  };
  constexpr int kLanes = D / 8, kRows = 32 / kLanes;  // lanes per row, rows per copy
  const int r0 = lane / kLanes, chunk = lane % kLanes;
  // Where a lane's 16 bytes go: 512 bytes on with every copy, the place in the
  // row turned by the rows passed (r0 and the steps share no bits).
  const uint32_t place = static_cast<uint32_t>(r0 * D * 2), turned = static_cast<uint32_t>((chunk ^ r0) << 4);
  auto place_of = [&](int i) { return place + i * 512 + (turned ^ (((i * kRows) & 7) << 4)); };
  const bool lane_on = chunk * 8 < hd;
  const int64_t lane_from = r0 * p.slot_stride + chunk * 8;
  const bool dense = p.slot_stride == D && hd == D;  // a page's rows of a head are one block
  const int64_t apart = static_cast<const CT*>(p.value) - static_cast<const CT*>(p.key);
  auto load_next = [&](int stage) {
    while (ld.it >= ld.end && ld.g < te) {  // on to the segment that holds the tile
      const Seg sg = segment(&ld.b, ld.g);
      ld.g = sg.next;
      ld.begin = ld.end;
      ld.end += sg.n;
      if (ld.it >= ld.end) continue;
      const Walk w = walk(ld.b);
      const int kvh = sg.pair / d.subs, last_page = w.hi >> shift;
      ld.list = d.pages ? d.pages + (static_cast<int64_t>(ld.b) * p.a.Hk + kvh) * d.count : nullptr;
      ld.head = kvh * p.head_stride + lane_from;
      ld.lo = w.lo;
      ld.hi = w.hi;
      ld.first = w.first + sg.lt;
      ld.e_first = ld.list ? 0 : w.lo >> shift;
      const int most = min(d.pages ? d.count : last_page + 1, last_page + 1);
      ld.e_end = min(static_cast<int>((static_cast<int64_t>(ld.first + sg.n) * C::kTile - 1) >> shift) + 1, most);
      ld.base = static_cast<int>((static_cast<int64_t>(ld.first + ld.it - ld.begin) * C::kTile) >> shift);
      look(ld.base + lane, &ld.index, &ld.page);
      look(ld.base + 32 + lane, &ld.index_next, &ld.page_next);
      // (one entry past a list of all pages: it has to be a negative one)
      if (ld.list) ld.e_end = min(ld.e_end, list_length(p, ld.list, min(d.count, last_page + 2), last_page, lane));
    }
    if (ld.it < ld.end) {
      const int64_t token = static_cast<int64_t>(ld.first + ld.it - ld.begin) * C::kTile;
      const int e = static_cast<int>(token >> shift), offset = static_cast<int>(token) & mask;
      if (e - ld.base >= 32) {
        ld.base += 32;
        ld.index = ld.index_next;
        ld.page = ld.page_next;
        look(ld.base + 32 + lane, &ld.index_next, &ld.page_next);
      }
      const uint32_t kst = ring + stage * C::kStageBytes;
#pragma unroll
      for (int u = 0; u < C::kGroups; ++u) {
        const int piece = (offset + u * 16) >> shift;  // pages of under a tile: the group's page within the tile
        const int index = __shfl_sync(0xffffffffu, ld.index, e - ld.base + piece);
        int page = __shfl_sync(0xffffffffu, ld.page, e - ld.base + piece);
        if (e + piece >= ld.e_end) page = kNowhere;
        if (static_cast<unsigned>(page) >= static_cast<unsigned>(p.page_count)) {
          if (page != kNowhere) report_error(p.a.error, TLA_ERR_PAGE);
          page = -1;
        }
        const int slot = (offset + u * 16) & mask;
        const int at = page < 0 ? kNowhere : (index << shift) + slot;
        if (lane == 0) meta[stage * C::kGroups + u] = at;
        const CT* k = static_cast<const CT*>(p.key) + (page * p.page_stride + slot * p.slot_stride + ld.head);
        const uint32_t dst = kst + u * 16 * D * 2;
        if (at >= ld.lo && at + 15 <= ld.hi) {  // (the same for the whole warp)
          if (dense) {
#pragma unroll
            for (int i = 0; i < 16 / kRows; ++i) {
              copy16(dst + place_of(i), k + i * kRows * D);
              copy16(dst + place_of(i) + C::kTileBytes, k + apart + i * kRows * D);
            }
          } else if (lane_on) {
#pragma unroll
            for (int i = 0; i < 16 / kRows; ++i) {
              copy16(dst + place_of(i), k);
              copy16(dst + place_of(i) + C::kTileBytes, k + apart);
              k += kRows * p.slot_stride;
            }
          }
        } else if (lane_on) {  // rows outside the range, and pages that are not there, as zeros
#pragma unroll 1
          for (int i = 0; i < 16 / kRows; ++i) {
            const int tok = at + r0 + i * kRows, bytes = tok >= ld.lo && tok <= ld.hi ? 16 : 0;
            const CT* from = bytes ? k + i * kRows * p.slot_stride : static_cast<const CT*>(p.key);
            copy16_or_zeros(dst + place_of(i), from, bytes);
            copy16_or_zeros(dst + place_of(i) + C::kTileBytes, bytes ? from + apart : from, bytes);
          }
        }
      }
    }
    copies_commit();
    ld.it += kWarps;
  };
#pragma unroll
  for (int s = 0; s < C::kStages; ++s) load_next(s);

  // ================================================================== products
  CT* q_s = reinterpret_cast<CT*>(smem + L.q);
  float* red = reinterpret_cast<float*>(smem + L.red);
  constexpr int kNt = TWO ? 2 : 1;  // column tiles of 8 query heads
  constexpr float kLift = kLiftOf<CT>;
  constexpr int kGroups = C::kGroups;
  const int g8 = lane >> 2, t4 = lane & 3;
  const int frag_row = (lane & 7) + ((lane >> 3) & 1) * 8;   // K as the left operand: token rows, then dimensions
  const int vfrag_row = (lane & 7) + (lane >> 4) * 8;        // V transposed: its tokens are the columns
  int it0 = 0, stage = 0;  // the share's tiles before this segment; the ring's oldest tile
  int b = 0;
  for (int g = tb; g < te;) {
    const Seg sg = segment(&b, g);
    if (sg.n == 0 && !d.cluster) {  // the share ends inside the pair's set-up units
      g = sg.next;
      continue;
    }
    const int kvh = sg.pair / d.subs, sub = sg.pair - kvh * d.subs;
    const int h0 = kvh * G + sub * rows, heads = min(rows, (kvh + 1) * G - h0);
    const Walk w = walk(b);
    const IO* q = static_cast<const IO*>(d.query) + (static_cast<int64_t>(b) * Hq + h0) * hd;
    // ---- the group's queries, 8 elements per thread and trip; rows past the group are zeros
    if constexpr (SPLIT) {
      for (int r = warp; r < 8 * kNt; r += kWarps) {
        float x[D / 32], top = 0.f;
#pragma unroll
        for (int e = 0; e < D / 32; ++e) {
          x[e] = r < heads && lane + 32 * e < hd ? q[r * hd + lane + 32 * e] : 0.f;
          top = fmaxf(top, fabsf(x[e]));
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        // largest element to [2^13, 2^14); a row of zeros or of values without an exponent stays
        int ex = static_cast<int>(__float_as_uint(top) >> 23) - 127;
        if (ex < -100 || ex > 127) ex = top == 0.f ? 0 : max(-100, min(ex, 127));
        ex -= 13;
        const float down = __uint_as_float(static_cast<uint32_t>(127 - ex) << 23);
#pragma unroll
        for (int e = 0; e < D / 32; ++e) {
          const float v = x[e] * down;
          const __half hi = __float2half_rz(v);  // (parts as pack2_cut and pack2_rest form them)
          q_s[r * (C::kQPitch / 2) + lane + 32 * e] = hi;
          q_s[(16 + r) * (C::kQPitch / 2) + lane + 32 * e] = __float2half_rn(fmaf(v, kUp, -__half2float(hi)));
        }
        if (lane == 0)  // (the row's padding)
          *reinterpret_cast<float*>(q_s + r * (C::kQPitch / 2) + D) = __uint_as_float(static_cast<uint32_t>(127 + ex) << 23);
      }
    } else {
      for (int i = tid; i < 8 * kNt * D / 8; i += 128) {
        const int r = i / (D / 8), c = i - r * (D / 8);
        const uint4 v = r < heads && c * 8 < hd ? *reinterpret_cast<const uint4*>(q + r * hd + c * 8)
                                                : make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(q_s + r * (C::kQPitch / 2) + c * 8) = v;
      }
    }
    __syncthreads();
    uint32_t qb[kNt][D / 16][2];
    uint32_t ql[kNt][SPLIT ? D / 16 : 1][2];
    float scale[kNt][2];
#pragma unroll
    for (int nt = 0; nt < kNt; ++nt) {
#pragma unroll
      for (int kk = 0; kk < D / 16; kk += 2) {  // 8 heads x 32 dimensions
        const uint32_t at = smem_u32(q_s) + (nt * 8 + (lane & 7)) * C::kQPitch + (2 * kk + (lane >> 3)) * 16;
        ldsm_x4(at, qb[nt][kk][0], qb[nt][kk][1], qb[nt][kk + 1][0], qb[nt][kk + 1][1]);
        if constexpr (SPLIT)
          ldsm_x4(at + 16 * C::kQPitch, ql[nt][kk][0], ql[nt][kk][1], ql[nt][kk + 1][0], ql[nt][kk + 1][1]);
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        scale[nt][e] = p.a.attn_scale * kLog2e;
        if constexpr (SPLIT)
          scale[nt][e] *= (1.f - 0x1p-23f) *  // (of the parts' kUp)
                          *reinterpret_cast<const float*>(q_s + (nt * 8 + 2 * t4 + e) * (C::kQPitch / 2) + D);
      }
    }

    // this thread's columns: heads nt * 8 + 2 * t4 + e; m is the weights' base
    float o[kNt][D / 16][4], m[kNt][2], l[kNt][2];
#pragma unroll
    for (int nt = 0; nt < kNt; ++nt) {
#pragma unroll
      for (int i = 0; i < D / 16; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
    }

    // ---- this warp's tiles of the segment
    const int it1 = it0 + sg.n;
    for (int it = it0 + ((warp - it0) & (kWarps - 1)); it < it1; it += kWarps) {
      copies_wait<C::kStages - 1>();
      __syncwarp();
      int at[kGroups];
      bool whole = true, any = false;
#pragma unroll
      for (int u = 0; u < kGroups; ++u) {
        at[u] = meta[stage * kGroups + u];
        whole = whole && at[u] >= w.lo && at[u] + 15 <= w.hi;
        any = any || (at[u] <= w.hi && at[u] + 15 >= w.lo);
      }
      if (any) {  // (the same for the whole warp)
        // S^T = K Q^T: tokens g8 and g8 + 8 of each group, columns 2 t4 and 2 t4 + 1
        float x[kGroups][kNt][4];
        const uint32_t kbase = ring + stage * C::kStageBytes;
#pragma unroll
        for (int u = 0; u < kGroups; ++u) {
#pragma unroll
          for (int nt = 0; nt < kNt; ++nt) x[u][nt][0] = x[u][nt][1] = x[u][nt][2] = x[u][nt][3] = 0.f;
        }
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const int chunk = 2 * kk + (lane >> 4);
#pragma unroll
          for (int u = 0; u < kGroups; ++u) {
            const int tok = u * 16 + frag_row;
            uint32_t a[4];
            ldsm_x4(kbase + tile_at<D>(tok, chunk), a[0], a[1], a[2], a[3]);
#pragma unroll
            for (int nt = 0; nt < kNt; ++nt) {
              mma_t<CT>(x[u][nt], a, qb[nt][kk][0], qb[nt][kk][1]);
              if constexpr (SPLIT) mma_t<CT>(x[u][nt], a, ql[nt][kk][0], ql[nt][kk][1]);
            }
          }
        }
        // mask + online softmax (log2 domain)
        uint32_t pb[kGroups][kNt][2], pl[kGroups][kNt][2];
#pragma unroll
        for (int nt = 0; nt < kNt; ++nt) {
          float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
          for (int u = 0; u < kGroups; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) x[u][nt][e] *= scale[nt][e & 1];
          if (!whole) {
#pragma unroll
            for (int u = 0; u < kGroups; ++u)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int tok = at[u] + g8 + (e >> 1) * 8;
                if (tok < w.lo || tok > w.hi) x[u][nt][e] = -INFINITY;
              }
          }
#pragma unroll
          for (int u = 0; u < kGroups; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) top[e & 1] = fmaxf(top[e & 1], x[u][nt][e]);
          float base[2], keep[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 4));
            top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 8));
            top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 16));
            top[e] = fmaxf(kLift > 0.f ? __fsub_ru(top[e], kLift) : top[e], m[nt][e]);
            base[e] = top[e] == -INFINITY ? 0.f : top[e];
            keep[e] = ex2(m[nt][e] - base[e]);
            m[nt][e] = top[e];
            l[nt][e] *= keep[e];
          }
#pragma unroll
          for (int u = 0; u < kGroups; ++u) {
            float pr[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              pr[e] = ex2(x[u][nt][e] - base[e & 1]);
              l[nt][e & 1] = fmaf(pr[e], kUp, l[nt][e & 1]);
            }
            const uint32_t p0 = pack2_cut<CT>(pr[0], pr[1]), p1 = pack2_cut<CT>(pr[2], pr[3]);
            pb[u][nt][0] = transpose8(p0);
            pb[u][nt][1] = transpose8(p1);
            pl[u][nt][0] = transpose8(pack2_rest<CT>(p0, pr[0], pr[1]));
            pl[u][nt][1] = transpose8(pack2_rest<CT>(p1, pr[2], pr[3]));
          }
          if (__any_sync(0xffffffffu, keep[0] != 1.f || keep[1] != 1.f)) {  // a maximum rose
#pragma unroll
            for (int i = 0; i < D / 16; ++i)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[nt][i][e] *= keep[e & 1];
          }
        }
        // O^T += V^T P^T: dimensions g8 and g8 + 8 of each 16
        const uint32_t vbase = kbase + C::kTileBytes;
#pragma unroll
        for (int u = 0; u < kGroups; ++u) {
          const int tok = u * 16 + vfrag_row;
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            const int chunk = 2 * i + ((lane >> 3) & 1);
            uint32_t a[4];
            ldsm_x4_t(vbase + tile_at<D>(tok, chunk), a[0], a[1], a[2], a[3]);
#pragma unroll
            for (int nt = 0; nt < kNt; ++nt) {
              mma_t<CT>(o[nt][i], a, pb[u][nt][0], pb[u][nt][1]);
              mma_t<CT>(o[nt][i], a, pl[u][nt][0], pl[u][nt][1]);
            }
          }
        }
      }
      __syncwarp();
      load_next(stage);
      stage = stage + 1 == C::kStages ? 0 : stage + 1;
    }
    it0 = it1;

    // ---- join the 4 warps' (m, l, O)
    float* rw = red + warp * rows * (D + 2);
#pragma unroll
    for (int nt = 0; nt < kNt; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float sum = l[nt][e];
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        const int r = nt * 8 + 2 * t4 + e;
        if (r < heads) {
          float* rr = rw + r * (D + 2);
          if (g8 == 0) {
            rr[0] = m[nt][e];
            rr[1] = sum;
          }
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            rr[2 + i * 16 + g8] = o[nt][i][e];
            rr[2 + i * 16 + 8 + g8] = o[nt][i][2 + e];
          }
        }
      }
    __syncthreads();
    const bool whole = d.cluster ? d.cluster == 1 : sg.lt == 0 && sg.n == sg.tiles;
    float* mine = d.cluster ? reinterpret_cast<float*>(smem + L.part)
                            : d.scratch + (static_cast<size_t>(cta) * 2 + (g == tb ? 0 : 1)) * rows * (D + 2);
    for (int i = tid; i < heads * (D / 2); i += kThreads) {  // two columns each
      const int r = i / (D / 2), c = i % (D / 2) * 2;
      float2 ml[kWarps];
#pragma unroll
      for (int k = 0; k < kWarps; ++k) ml[k] = *reinterpret_cast<const float2*>(red + (k * rows + r) * (D + 2));
      const float top = fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x)), base = top == -INFINITY ? 0.f : top;
      float sum = 0.f, v0 = 0.f, v1 = 0.f;
#pragma unroll
      for (int k = 0; k < kWarps; ++k) {
        const float2 x = *reinterpret_cast<const float2*>(red + (k * rows + r) * (D + 2) + 2 + c);
        const float f = ex2(ml[k].x - base);
        sum += ml[k].y * f;
        v0 += x.x * f;
        v1 += x.y * f;
      }
      if (whole) {
        const float inv = inverse(sum);
        if (c < hd) store_out<IO>(d, (static_cast<int64_t>(b) * Hq + h0 + r) * hd + c, v0, inv);
        if (c < hd) store_out<IO>(d, (static_cast<int64_t>(b) * Hq + h0 + r) * hd + c + 1, v1, inv);
      } else if (d.cluster ||
                 TLA_IN_BOUNDS(mine - d.scratch + (r + 1) * (D + 2) - 1, d.scratch_floats, p.a.error)) {
        *reinterpret_cast<float2*>(mine + r * (D + 2) + 2 + c) = make_float2(v0, v1);
        if (c == 0) *reinterpret_cast<float2*>(mine + r * (D + 2)) = make_float2(top, sum);
      }
    }
    __syncthreads();  // red and q_s are free for the next segment
    g = sg.next;
  }

  if (d.cluster > 1) {  // join the cluster's triples, a part of the columns in each of its CTAs
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    const int kvh = only.pair / d.subs, sub = only.pair - kvh * d.subs;
    const int h0 = kvh * G + sub * rows, heads = min(rows, (kvh + 1) * G - h0);
    float* part = reinterpret_cast<float*>(smem + L.part);
    for (int i = cluster.block_rank() * kThreads + tid; i < heads * (D / 2); i += d.cluster * kThreads) {
      const int r = i / (D / 2), c = i % (D / 2) * 2;
      if (c >= hd) continue;
      float2 ml[kMaxCluster], x[kMaxCluster];
      float top = -INFINITY;
#pragma unroll
      for (int k = 0; k < kMaxCluster; ++k) {
        ml[k] = make_float2(-INFINITY, 0.f);
        x[k] = make_float2(0.f, 0.f);
        if (k < d.cluster) {
          const float* of = cluster.map_shared_rank(part, k) + r * (D + 2);
          ml[k] = *reinterpret_cast<const float2*>(of);
          x[k] = *reinterpret_cast<const float2*>(of + 2 + c);
        }
      }
#pragma unroll
      for (int k = 0; k < kMaxCluster; ++k) top = fmaxf(top, ml[k].x);
      const float base = top == -INFINITY ? 0.f : top;
      float sum = 0.f, v0 = 0.f, v1 = 0.f;
#pragma unroll
      for (int k = 0; k < kMaxCluster; ++k) {
        const float f = ex2(ml[k].x - base);
        sum += ml[k].y * f;
        v0 += x[k].x * f;
        v1 += x[k].y * f;
      }
      const float inv = inverse(sum);
      store_out<IO>(d, (static_cast<int64_t>(only_b) * Hq + h0 + r) * hd + c, v0, inv);
      store_out<IO>(d, (static_cast<int64_t>(only_b) * Hq + h0 + r) * hd + c + 1, v1, inv);
    }
    cluster.sync();  // the others may still read this CTA's triple
  }
}

// Joins the triples of the pairs that several CTAs shared: a block per (pair,
// query head). It recomputes the shares from the positions, which it may read
// before the first kernel has finished: that kernel only starts its successor
// once its own wait for what came before is over.
constexpr int kJoinWarps = 4;
template <int D, typename IO>
__global__ void __launch_bounds__(kJoinWarps * 32) paged_decode_join_kernel(const __grid_constant__ DecodeParams d,
                                                                           int launch_grid) {
  constexpr int kPer = D / 32, kBatch = 8;
  __shared__ int prefix[kMaxBatch + 1];
  __shared__ int slot_of[kMaxGrid];
  __shared__ float red[2][kJoinWarps];
  __shared__ float row_s[kJoinWarps][D];
  griddep_launch_dependents();
  const PagedArgs& p = d.p;
  const int G = p.a.G, pairs = p.a.Hk * d.subs;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int b = blockIdx.x / p.a.Hq, h = blockIdx.x - b * p.a.Hq;
  const int kvh = h / G, sub = (h - kvh * G) / d.rows, r = (h - kvh * G) - sub * d.rows;
  for (int i = tid; i < p.batch; i += kJoinWarps * 32) prefix[i + 1] = units_of<D>(d, p.positions[i]);
  if (tid == 0) prefix[0] = 0;
  __syncthreads();
  if (warp == 0) scan_prefix(prefix, p.batch, lane);
  __syncthreads();
  const int total = prefix[p.batch], grid = effective_grid(total, launch_grid, d.small_grid);
  const bool held = prefix[b + 1] != prefix[b];
  int c0 = 0, c1 = 0;
  if (held) {
    const int per = (prefix[b + 1] - prefix[b]) / pairs, start = prefix[b] + (kvh * d.subs + sub) * per;
    c0 = cta_of(start + Cfg<D>::kSetup, total, grid);
    c1 = cta_of(start + per - 1, total, grid);
    // a CTA whose share begins at or after the pair's first unit holds it as its first segment
    for (int c = c0 + tid; c <= c1; c += kJoinWarps * 32) {
      const int cb = cta_begin(c, total, grid);
      slot_of[c - c0] = cta_begin(c + 1, total, grid) == cb ? -1 : 2 * c + (cb >= start ? 0 : 1);
    }
  }
  __syncthreads();
  griddep_wait();
  if (c0 == c1) return;  // one CTA held the whole pair, or there is none
  const int n = c1 - c0 + 1;
  const bool alone = n <= kBatch;  // few triples: one warp joins them without the others
  if (alone && warp != 0) return;
  const int warps = alone ? 1 : kJoinWarps;
  float top = -INFINITY, sum = 0.f, acc[kPer];
#pragma unroll
  for (int e = 0; e < kPer; ++e) acc[e] = 0.f;
  for (int k = warp; k < n; k += kBatch * warps) {
    float mk[kBatch], lk[kBatch], v[kBatch][kPer];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int at = k + u * warps;
      int slot = at < n ? slot_of[at] : -1;
      if (slot >= 0 && !TLA_IN_BOUNDS((static_cast<long long>(slot) + 1) * d.rows * (D + 2) - 1, d.scratch_floats,
                                      p.a.error))
        slot = -1;
      mk[u] = -INFINITY;
      lk[u] = 0.f;
#pragma unroll
      for (int e = 0; e < kPer; ++e) v[u][e] = 0.f;
      if (slot >= 0) {
        const float* t = d.scratch + (static_cast<size_t>(slot) * d.rows + r) * (D + 2);
        mk[u] = t[0];
        lk[u] = t[1];
#pragma unroll
        for (int e = 0; e < kPer; ++e) v[u][e] = t[2 + lane + 32 * e];
      }
    }
    float high = top;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) high = fmaxf(high, mk[u]);
    const float base = high == -INFINITY ? 0.f : high, keep = ex2(top - base);
    sum *= keep;
#pragma unroll
    for (int e = 0; e < kPer; ++e) acc[e] *= keep;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const float f = ex2(mk[u] - base);
      sum += lk[u] * f;
#pragma unroll
      for (int e = 0; e < kPer; ++e) acc[e] += v[u][e] * f;
    }
    top = high;
  }
  if (alone) {
#pragma unroll
    for (int e = 0; e < kPer; ++e)
      if (lane + 32 * e < p.a.D)
        store_out<IO>(d, static_cast<int64_t>(blockIdx.x) * p.a.D + lane + 32 * e, acc[e], inverse(sum));
    return;
  }
  if (lane == 0) {
    red[0][warp] = top;
    red[1][warp] = sum;
  }
#pragma unroll
  for (int e = 0; e < kPer; ++e) row_s[warp][lane + 32 * e] = acc[e];
  __syncthreads();
  float high = red[0][0];
#pragma unroll
  for (int w = 1; w < kJoinWarps; ++w) high = fmaxf(high, red[0][w]);
  const float base = high == -INFINITY ? 0.f : high;
  for (int c = tid; c < p.a.D; c += kJoinWarps * 32) {
    float all = 0.f, v = 0.f;
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) {
      const float f = ex2(red[0][w] - base);
      all += red[1][w] * f;
      v += row_s[w][c] * f;
    }
    store_out<IO>(d, static_cast<int64_t>(blockIdx.x) * p.a.D + c, v, inverse(all));
  }
}

// Two CTAs per SM by registers (the launch bounds), if shared memory holds two
// (228 KB, 1 KB of it reserved per CTA).
int ctas_per_sm(int smem) {
  const int n = 228 * 1024 / (smem + 1024);
  return n < kCtasPerSm ? n : kCtasPerSm;
}

template <int D, typename CT, bool SPLIT, bool TWO>
cudaError_t launch_t(const tla_paged* P, DecodeParams& d, cudaStream_t stream) {
  using IO = typename std::conditional<SPLIT, float, CT>::type;
  auto kernel = paged_decode_kernel<D, CT, SPLIT, TWO>;
  const int smem = smem_layout<D>(d.rows, d.cluster ? 0 : d.p.batch, SPLIT).total;
  if (d.cluster) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(d.p.batch) * P->base.Hk * d.subs * d.cluster);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = d.cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = d.cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, d);
  }
  const int grid = ctas_per_sm(smem) * P->base.ctx->sm_count;
  d.small_grid = P->base.ctx->sm_count;
  const cudaError_t e = launch_pdl(kernel, grid, kThreads, smem, stream, d);
  if (e != cudaSuccess) return e;
  return launch_pdl(paged_decode_join_kernel<D, IO>, static_cast<unsigned>(d.p.batch) * P->base.Hq, kJoinWarps * 32, 0,
                    stream, d, grid);
}

template <typename F>
auto by_width(const tla_paged* P, F f) {
  const int D = P->base.D;
  if (D <= 64) return f(std::integral_constant<int, 64>());
  if (D <= 128) return f(std::integral_constant<int, 128>());
  return f(std::integral_constant<int, 256>());
}

// What launches of an instance need to have been set for it: the shared memory
// of the layer's largest calls, and clusters of up to 16 (*most: 8 where the
// device does not run those).
template <int D, typename CT, bool SPLIT, bool TWO>
cudaError_t configure_t(int rows, int max_batch, int* most) {
  const void* k = reinterpret_cast<const void*>(paged_decode_kernel<D, CT, SPLIT, TWO>);
  const int smem = smem_layout<D>(rows, max_batch < kMaxBatch ? max_batch : kMaxBatch, SPLIT).total;
  cudaError_t e = raise_smem_limit(k, smem);
  if (e != cudaSuccess) return e;
  return large_cluster(k, kThreads, smem_layout<D>(rows, 0, SPLIT).total, most);
}
// f(an instance of the kernel) for the layer's types and `rows` query heads per
// group (256 wide there are groups of at most 8: two column tiles of O would not
// fit the registers).
template <typename CT, bool SPLIT, bool TWO>
struct Instance {
  using Type = CT;
  static constexpr bool kSplit = SPLIT, kTwo = TWO;
};
template <int D, typename F>
cudaError_t by_instance(const tla_paged* P, int rows, F f) {
  if constexpr (D < 256)
    if (rows > 8) {
      if (P->io == kFp32) return f(Instance<__half, true, true>());
      if (P->kept == kBf16) return f(Instance<__nv_bfloat16, false, true>());
      return f(Instance<__half, false, true>());
    }
  if (P->io == kFp32) return f(Instance<__half, true, false>());
  if (P->kept == kBf16) return f(Instance<__nv_bfloat16, false, false>());
  return f(Instance<__half, false, false>());
}

int subgroups(const tla_paged* P) {
  const int most = P->base.D > 128 ? 8 : 16;
  return (P->base.G + most - 1) / most;
}
int subgroup_rows(const tla_paged* P) {
  const int s = subgroups(P);
  return (P->base.G + s - 1) / s;
}

}  // namespace

// The tensor-core path takes 16-bit pages of 16 tokens and up (16 tokens lie in
// one page), head_dim a multiple of 8 and pools with rows on 16-byte boundaries;
// float32 activations only over float16 pages (two bfloat16 parts would carry
// 16 bits).
cudaError_t paged_decode_configure(tla_paged* P) {
  P->fast = P->wide && P->kept != kFp32 && (P->io != kFp32 || P->kept == kFp16) && P->pool.page_size >= 16 &&
            kCtasPerSm * P->base.ctx->sm_count <= kMaxGrid;
  if (!P->fast) return cudaSuccess;
  const int rows = subgroup_rows(P);
  return by_width(P, [&](auto w) {
    constexpr int D = decltype(w)::value;
    return by_instance<D>(P, rows, [&](auto i) {
      using I = decltype(i);
      return configure_t<D, typename I::Type, I::kSplit, I::kTwo>(rows, P->base.max_batch, &P->decode_cluster);
    });
  });
}

// The most tiles that a pair of this call can have.
long long most_tiles(const PagedArgs& p, int count) {
  const int kTile = p.a.D <= 64 ? Cfg<64>::kTile : Cfg<128>::kTile;
  long long tokens = p.capacity, tiles = (tokens + kTile - 1) / kTile;
  if (count > 0) {
    const long long listed = ((static_cast<long long>(count) << p.page_shift) + kTile - 1) / kTile;
    tiles = listed < tiles ? listed : tiles;
  } else if (p.a.sliding > 0) {
    const long long seen = (p.a.sliding - 2LL) / kTile + 2;
    tiles = seen < tiles ? seen : tiles;
  }
  return tiles;
}

// CTAs per pair when a cluster takes it, 0 when the pairs' tiles are cut into
// shares. A cluster joins its triples itself: one launch, no workspace, only
// its own sequence's position to wait for. It gets a CTA per four tiles, up to
// 16 (8 above head_dim 128) and up to two CTAs per SM in all. Shares balance
// unequal lengths and fill every SM; they win where a CTA of a cluster would get
// many tiles. Measured (shares / cluster, us; 4 query heads for each of 8 kv
// heads; * what the rule takes):
//   head_dim 64:  1 x 1025 tokens 7.0 / 5.7*, 1 x 8193 8.6* / 9.4, 8 x 4097 17.8 / 16.5*,
//                 64 x 1025 35.1 / 29.4*
//   head_dim 128: 1 x 1025 8.6 / 7.0*, 1 x 8193 12.6* / 12.8, 8 x 2049 17.7 / 16.5*,
//                 8 x 4097 27.7* / 25.8, 64 x 1025 53.1* / 47.2
//   head_dim 256: 1 x 1025 9.5 / 9.0*, 1 x 2049 9.8 / 11.0*, 1 x 4097 13.3* / 15.5, 8 x 4097 48.9* / 46.4
// and of lengths from a sixteenth up:
//   head_dim 64:  16 x 2049 12.6 / 13.1*, 64 x 2049 30.8* / 28.1, 64 x 4097 45.4* / 47.6
//   head_dim 128: 16 x 2049 16.3* / 19.5, 64 x 2049 45.6* / 44.8, 64 x 4097 75.2* / 80.1
// Above head_dim 128 an SM holds one CTA, and clusters of 16 leave a GPC's other
// SMs idle: 1 x 1025, 2049 and 4097 took 15.2, 17.3 and 22.0 us in them.
int cluster_size(const tla_paged* P, const PagedArgs& p, int count) {
  const long long tiles = most_tiles(p, count), pairs = static_cast<long long>(p.batch) * p.a.Hk * subgroups(P);
  const int sms = P->base.ctx->sm_count;
  const int per_sm = p.a.D > 128 ? 1 : kCtasPerSm;
  const int most = p.a.D > 128 && P->decode_cluster > 8 ? 8 : P->decode_cluster;
  int n = 1;
  while (n < most && tiles > 4 * n && pairs * n * 2 <= per_sm * sms) n *= 2;
  return tiles <= (pairs * n > sms ? 40 : 20) * n ? n : 0;
}

// Whether a call's pairs make a grid, or its shares can be cut: the batch's
// table fits shared memory and its tiles are counted in 32 bits.
bool paged_decode_takes(const tla_paged* P, const PagedArgs& p, int count) {
  if (!P->fast) return false;
  const long long pairs = static_cast<long long>(p.a.Hk) * subgroups(P) * p.batch;
  if (cluster_size(P, p, count) > 0) return pairs < (1LL << 26);
  return p.batch <= kMaxBatch && (most_tiles(p, count) + 16) * pairs < (1LL << 31);
}

size_t paged_decode_workspace(const tla_paged* P, const PagedArgs& p, int count) {
  if (cluster_size(P, p, count) > 0) return 0;
  const int width = by_width(P, [](auto w) { return decltype(w)::value; });
  return static_cast<size_t>(kCtasPerSm) * P->base.ctx->sm_count * 2 * subgroup_rows(P) * (width + 2) * sizeof(float);
}

cudaError_t launch_paged_decode(const tla_paged* P, const PagedArgs& p, const void* query, const int32_t* pages,
                                int count, const void* gate, void* out, void* workspace, cudaStream_t stream) {
  DecodeParams d;
  d.p = p;
  d.query = query;
  d.pages = pages;
  d.gate = gate;
  d.out = out;
  d.scratch = static_cast<float*>(workspace);
  d.scratch_floats = static_cast<long long>(paged_decode_workspace(P, p, count) / sizeof(float));
  d.count = count;
  d.subs = subgroups(P);
  d.rows = subgroup_rows(P);
  d.small_grid = 0;
  d.cluster = cluster_size(P, p, count);
  return by_width(P, [&](auto w) {
    constexpr int D = decltype(w)::value;
    return by_instance<D>(P, d.rows, [&](auto i) {
      using I = decltype(i);
      return launch_t<D, typename I::Type, I::kSplit, I::kTwo>(P, d, stream);
    });
  });
}

}  // namespace tla
