// Persistent split-KV decode over a paged cache (sm_100a): 16-bit pages,
// head_dim 64 or 128, pages of 16 tokens and up.
//
//   o = sum_t 2^(x_t - m) v_t / sum_t 2^(x_t - m),  x_t = log2(e) scale q.k_t
//
// Each K and V element is read once and used by the group's query heads, about
// 2 G operations per byte: memory bounds it, so the kernel's shape follows the
// reads. A (sequence, kv head) pair's tokens are cut into tiles (64 tokens at
// head_dim 64, 32 at 128: 16 KB of K and V), and the tiles of all pairs into
// equal contiguous shares, one per resident CTA, whatever the sequences'
// lengths; a share may begin and end inside a pair. A producer warp walks the
// share's pages: its lanes look up 32 table entries at a time, one window
// ahead, and start one TMA box per page piece of a tile (five-dimensional
// tensor maps: any order and padding of pages, heads and slots, as long as the
// strides are multiples of 16 bytes) into a ring of stages. Four consumer warps
// take the tiles in turn, each a whole tile by itself, so that a tile's chain
// of products, maximum, exponentials and products again is four deep in flight
// per CTA and needs no barrier between warps. 16 tokens always lie in one
// page: a page's end inside a tile, a page that is not in the pool and the
// window's edges are decided per 16 tokens from their first position, which
// the producer leaves beside the stage.
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
// float32 activations over float16 pages: each query row is scaled by a power
// of two and split into two float16 parts, and so is each weight; with both
// parts multiplied the products carry 22 bits, and the output keeps float32's
// use for its caller. K and V are exact as stored.
#include <math.h>

#include <type_traits>

#include "paged.cuh"

namespace tla {

namespace {

constexpr int kConsumerWarps = 4;
constexpr int kThreads = (kConsumerWarps + 1) * 32;
constexpr int kMaxBatch = 1024;  // prefix table in shared memory
constexpr int kCtasPerSm = 2;
constexpr int kMaxGrid = 1024;   // segment table of the joining kernel
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kNowhere = -(1 << 30);  // first position of 16 tokens that take no part

#ifndef STG
#define STG 4
#endif
#ifndef TILE64
#define TILE64 64
#endif
#ifndef TILE128
#define TILE128 32
#endif
#ifndef SETUP64
#define SETUP64 4
#endif
#ifndef SETUP128
#define SETUP128 4
#endif
template <int D>
struct Cfg {
  static constexpr int kTile = D == 64 ? TILE64 : TILE128;
  static constexpr int kGroups = kTile / 16;
  static constexpr int kStages = STG;      // a multiple of the consumer warps: a stage is always the same warp's
  static constexpr int kHalves = D / 64;  // 128-byte rows per cache row
  static constexpr int kTileBytes = kTile * kHalves * 128;
  static constexpr int kStageBytes = 2 * kTileBytes;
  static constexpr int kQPitch = D * 2 + 16;
  // A pair costs its query set-up and its epilogue besides its tiles: counted
  // as this many tiles when the shares are cut.
  static constexpr int kSetup = D == 64 ? SETUP64 : SETUP128;
};

struct DecodeParams {
  CUtensorMap tmap_k;
  CUtensorMap tmap_v;
  PagedArgs p;
  const void* query;
  const int32_t* pages;  // null, or [batch][Hk][count]
  const void* gate;
  void* out;
  float* scratch;  // [grid][2][rows][D + 2]
  int count;
  int subs;        // groups of up to 16 query heads per kv head
  int rows;        // query heads per such group, the last one's may be fewer
  int small_grid;
  int whole;       // every pair goes to one CTA: nothing is joined
};

struct SmemLayout {
  int stages, q, red, meta, prefix, bars, flags, total;
};
template <int D>
__host__ __device__ inline SmemLayout smem_layout(int rows, int batch, bool split) {
  using C = Cfg<D>;
  SmemLayout s;
  int off = 0;
  s.stages = off;
  off += C::kStages * C::kStageBytes;
  s.q = off;
  off += (split ? 2 : 1) * 16 * C::kQPitch;
  s.red = off;
  off += kConsumerWarps * rows * (D + 2) * 4;
  off = (off + 15) & ~15;
  s.meta = off;
  off += C::kStages * 16;
  s.prefix = off;
  off += (2 * batch + 2) * 4;  // unit prefix, then positions
  off = (off + 7) & ~7;
  s.bars = off;
  off += 2 * C::kStages * 8;
  s.flags = off;
  off += 16;
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
__device__ __forceinline__ int cta_begin(int c, int total, int grid) {
  return static_cast<int>(static_cast<long long>(c) * total / grid);
}
// Largest c with cta_begin(c) <= g.
__device__ __forceinline__ int cta_of(int g, int total, int grid) {
  int c = static_cast<int>(static_cast<long long>(g) * grid / total);
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

// The first pair that starts at or after unit g.
__device__ __forceinline__ int next_pair(const int* prefix, int batch, int pairs, int g) {
  if (g >= prefix[batch]) return prefix[batch];
  int b = 0, n = batch;  // prefix[b] <= g < prefix[b + n]
  while (n > 1) {
    const int half = n / 2;
    if (prefix[b + half] <= g) {
      b += half;
      n -= half;
    } else {
      n = half;
    }
  }
  const int per = (prefix[b + 1] - prefix[b]) / pairs;
  return prefix[b] + (g - prefix[b] + per - 1) / per * per;
}

__device__ __forceinline__ void tma_load_5d(void* dst, const CUtensorMap* map, uint64_t* bar, int slot, int head,
                                            int page) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %2, %3, %4, %5}], "
      "[%6];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(slot), "r"(head), "r"(page), "r"(smem_u32(bar))
      : "memory");
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
// What pack_half2 rounded away of (lo, hi), as a pair of its own.
__device__ __forceinline__ uint32_t pack_rest(uint32_t packed, float lo, float hi) {
  const float2 f = __half22float2(*reinterpret_cast<__half2*>(&packed));
  return pack_half2(lo - f.x, hi - f.y);
}

// An 8 x 8 matrix of 16-bit values, a row pair of which each lane holds, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

template <typename IO>
__device__ __forceinline__ void store_out(const DecodeParams& d, int64_t i, float v) {
  if (d.gate) v = v * (1.f / (1.f + expf(-to_f32(static_cast<const IO*>(d.gate)[i]))));  // math.ts:271-273
  static_cast<IO*>(d.out)[i] = from_f32<IO>(v);
}

// SPLIT: float32 activations over float16 pages. TWO: more than 8 query heads per group.
template <int D, typename CT, bool SPLIT, bool TWO>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) paged_decode_kernel(const __grid_constant__ DecodeParams d) {
  using C = Cfg<D>;
  using IO = typename std::conditional<SPLIT, float, CT>::type;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const PagedArgs& p = d.p;
  const int Hq = p.a.Hq, G = p.a.G, pairs = p.a.Hk * d.subs, rows = d.rows;
  const SmemLayout L = smem_layout<D>(rows, p.batch, SPLIT);
  uint8_t* stages = smem + L.stages;
  int* prefix = reinterpret_cast<int*>(smem + L.prefix);
  int* spos = prefix + p.batch + 1;
  int* meta = reinterpret_cast<int*>(smem + L.meta);  // [stage][4]: first position of each 16 tokens of its tile
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L.bars);
  uint64_t* empty = full + C::kStages;
  volatile int* flags = reinterpret_cast<volatile int*>(smem + L.flags);  // [0] a wait gave up
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, cta = blockIdx.x;
  if (tid == 0) {
    flags[0] = 0;
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    fence_mbar_init();
    prefix[0] = 0;
    tma_prefetch(&d.tmap_k);
    tma_prefetch(&d.tmap_v);
  }
  griddep_wait();
  griddep_launch_dependents();
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
      for (int i = tid; i < Hq * D; i += kThreads)
        static_cast<IO*>(d.out)[static_cast<int64_t>(b) * Hq * D + i] = from_f32<IO>(0.f);
  const int grid = effective_grid(total, gridDim.x, d.small_grid);
  if (total == 0 || cta >= grid) return;
  int tb = cta_begin(cta, total, grid), te = cta_begin(cta + 1, total, grid);
  if (d.whole) {
    tb = next_pair(prefix, p.batch, pairs, tb);
    te = next_pair(prefix, p.batch, pairs, te);
  }
  if (tb >= te) return;
  const int shift = p.page_shift, mask = (1 << shift) - 1;

  if (warp == kConsumerWarps) {
    // ================================================================ producer
    constexpr int kTile = C::kTile;
    const int boxes = max(1, kTile >> shift);  // per tile, K or V
    const int box_rows = kTile / boxes, box_bytes = C::kTileBytes / boxes;
    uint32_t it = 0;
    int b = 0;
    for (int g = tb; g < te;) {
      while (prefix[b + 1] <= g) ++b;
      const Seg sg = seg_at<D>(prefix, b, pairs, g, te);
      g = sg.next;
      if (sg.n == 0) continue;
      const int kvh = sg.pair / d.subs;
      const Walk w = walk_of<D>(d, spos[b]);
      const int32_t* list = d.pages ? d.pages + (static_cast<int64_t>(b) * p.a.Hk + kvh) * d.count : nullptr;
      const int last_page = w.hi >> shift;
      // entries of the table (or the list) that this share walks
      const int t_begin = w.first + sg.lt, t_end = t_begin + sg.n;
      const int e_begin = static_cast<int>((static_cast<int64_t>(t_begin) * kTile) >> shift);
      int e_end = static_cast<int>((static_cast<int64_t>(t_end) * kTile - 1) >> shift) + 1;
      e_end = min(e_end, list ? list_length(p, list, min(d.count, last_page + 1), last_page, lane) : last_page + 1);
      const int e_first = list ? 0 : w.lo >> shift;
      // a lane's entry of a window of 32: the page's index in the sequence and its place in the pool
      auto look = [&](int e, int* index, int* page) {
        const bool in = e >= e_first && e < e_end;
        *index = !in ? 0 : list ? list[e] : e;
        *page = in ? pool_page(p, b, *index) : -1;
      };
      int base = e_begin, index, page, index_next, page_next;
      look(base + lane, &index, &page);
      look(base + 32 + lane, &index_next, &page_next);
      for (int t = t_begin; t < t_end; ++t, ++it) {
        const int s = it % C::kStages;
        const uint32_t ph = (it / C::kStages) & 1u;
        const int64_t token = static_cast<int64_t>(t) * kTile;
        const int e = static_cast<int>(token >> shift), offset = static_cast<int>(token) & mask;
        if (e - base >= 32) {
          base += 32;
          index = index_next;
          page = page_next;
          look(base + 32 + lane, &index_next, &page_next);
        }
        const int piece = lane % boxes;  // lanes 0..boxes-1 load K, the next V
        const int my_page = __shfl_sync(0xffffffffu, page, e - base + piece);
        const int group_piece = lane * 16 / box_rows;  // first lanes: the tile's groups of 16 tokens
        const int g_index = __shfl_sync(0xffffffffu, index, e - base + (lane < C::kGroups ? group_piece : 0));
        const int g_page = __shfl_sync(0xffffffffu, page, e - base + (lane < C::kGroups ? group_piece : 0));
        const int loaded = __popc(__ballot_sync(0xffffffffu, lane < boxes && my_page >= 0));
        const bool go = !flags[0] && mbar_wait(&empty[s], ph ^ 1u, p.a.error);
        if (__any_sync(0xffffffffu, !go)) {
          flags[0] = 1;
          continue;
        }
        if (lane < C::kGroups)
          meta[s * 4 + lane] = g_page < 0 ? kNowhere : (g_index << shift) + offset + lane * 16 - group_piece * box_rows;
        __syncwarp();
        if (lane == 0) mbar_arrive_expect_tx(&full[s], 2 * loaded * box_bytes);
        __syncwarp();
        if (lane < 2 * boxes && my_page >= 0)
          tma_load_5d(stages + s * C::kStageBytes + (lane < boxes ? 0 : C::kTileBytes) + piece * box_bytes,
                      lane < boxes ? &d.tmap_k : &d.tmap_v, &full[s], offset, kvh, my_page);
      }
    }
    // Do not leave the CTA with copies in flight.
    const uint32_t first = it > static_cast<uint32_t>(C::kStages) ? it - C::kStages : 0u;
    for (uint32_t i = first; i < it; ++i)
      if (!flags[0]) mbar_wait(&full[i % C::kStages], (i / C::kStages) & 1u, p.a.error);
    return;
  }

  // ================================================================== consumers
  CT* q_s = reinterpret_cast<CT*>(smem + L.q);
  float* red = reinterpret_cast<float*>(smem + L.red);
  constexpr int kNt = TWO ? 2 : 1;  // column tiles of 8 query heads
  constexpr int kGroups = C::kGroups;
  const int g8 = lane >> 2, t4 = lane & 3;
  const int frag_row = (lane & 7) + ((lane >> 3) & 1) * 8;   // K as the left operand: token rows, then dimensions
  const int vfrag_row = (lane & 7) + (lane >> 4) * 8;        // V transposed: its tokens are the columns
  uint32_t it0 = 0;  // the share's tiles before this segment
  int b = 0;
  for (int g = tb; g < te;) {
    while (prefix[b + 1] <= g) ++b;
    const Seg sg = seg_at<D>(prefix, b, pairs, g, te);
    if (sg.n == 0) {  // the share ends inside the pair's set-up units
      g = sg.next;
      continue;
    }
    const int kvh = sg.pair / d.subs, sub = sg.pair - kvh * d.subs;
    const int h0 = kvh * G + sub * rows, heads = min(rows, (kvh + 1) * G - h0);
    const Walk w = walk_of<D>(d, spos[b]);
    const IO* q = static_cast<const IO*>(d.query) + (static_cast<int64_t>(b) * Hq + h0) * D;
    // ---- the group's queries, 8 elements per thread and trip; rows past the group are zeros
    if constexpr (SPLIT) {
      for (int r = warp; r < 8 * kNt; r += kConsumerWarps) {
        float x[D / 32], top = 0.f;
#pragma unroll
        for (int e = 0; e < D / 32; ++e) {
          x[e] = r < heads ? q[r * D + lane + 32 * e] : 0.f;
          top = fmaxf(top, fabsf(x[e]));
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        // largest element to [1, 2); a row of zeros or of values without an exponent stays
        int ex = static_cast<int>(__float_as_uint(top) >> 23) - 127;
        if (ex < -100 || ex > 120) ex = top == 0.f ? 0 : max(-100, min(ex, 120));
        const float down = __uint_as_float(static_cast<uint32_t>(127 - ex) << 23);
#pragma unroll
        for (int e = 0; e < D / 32; ++e) {
          const float v = x[e] * down;
          const __half hi = __float2half_rn(v);
          q_s[r * (C::kQPitch / 2) + lane + 32 * e] = hi;
          q_s[(16 + r) * (C::kQPitch / 2) + lane + 32 * e] = __float2half_rn(v - __half2float(hi));
        }
        if (lane == 0)  // (the row's padding)
          *reinterpret_cast<float*>(q_s + r * (C::kQPitch / 2) + D) = __uint_as_float(static_cast<uint32_t>(127 + ex) << 23);
      }
    } else {
      for (int i = tid; i < 8 * kNt * D / 8; i += 128) {
        const int r = i / (D / 8), c = i - r * (D / 8);
        const uint4 v = r < heads ? reinterpret_cast<const uint4*>(q)[i] : make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(q_s + r * (C::kQPitch / 2) + c * 8) = v;
      }
    }
    named_barrier_sync(1, 128);
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
          scale[nt][e] *= *reinterpret_cast<const float*>(q_s + (nt * 8 + 2 * t4 + e) * (C::kQPitch / 2) + D);
      }
    }

    // this thread's columns: heads nt * 8 + 2 * t4 + e
    float o[kNt][D / 16][4], m[kNt][2], l[kNt][2];
#pragma unroll
    for (int nt = 0; nt < kNt; ++nt) {
#pragma unroll
      for (int i = 0; i < D / 16; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
    }

    // ---- this warp's tiles of the segment
    const uint32_t it1 = it0 + sg.n;
    for (uint32_t it = it0 + ((warp - it0) & (kConsumerWarps - 1)); it < it1; it += kConsumerWarps) {
      const int s = it % C::kStages;
      const uint32_t ph = (it / C::kStages) & 1u;
      if (!flags[0] && !mbar_wait(&full[s], ph, p.a.error)) flags[0] = 1;
      __syncwarp();
      uint8_t* kst = stages + s * C::kStageBytes;
      uint8_t* vst = kst + C::kTileBytes;
      int at[kGroups];
      bool whole = !flags[0], any = false;
#pragma unroll
      for (int u = 0; u < kGroups; ++u) {
        at[u] = meta[s * 4 + u];
        whole = whole && at[u] >= w.lo && at[u] + 15 <= w.hi;
        any = any || (at[u] <= w.hi && at[u] + 15 >= w.lo);
      }
      whole = __all_sync(0xffffffffu, whole);
      if (__all_sync(0xffffffffu, any && !flags[0])) {
        if (!whole) {
          // Slots outside the range, and pieces that were not loaded, may hold
          // anything: their weights are 0, and their values must be finite for
          // 0 v to be 0.
          for (int i = lane; i < C::kTile * C::kHalves * 8; i += 32) {
            const int r = i / (C::kHalves * 8), tok = meta[s * 4 + r / 16] + r % 16;
            if (tok < w.lo || tok > w.hi) *reinterpret_cast<uint4*>(vst + i * 16) = make_uint4(0, 0, 0, 0);
          }
          __syncwarp();
        }
        // S^T = K Q^T: tokens g8 and g8 + 8 of each group, columns 2 t4 and 2 t4 + 1
        float x[kGroups][kNt][4];
        const uint32_t kbase = smem_u32(kst);
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
            ldsm_x4(kbase + sw128(tok * C::kHalves + (chunk >> 3), chunk & 7), a[0], a[1], a[2], a[3]);
#pragma unroll
            for (int nt = 0; nt < kNt; ++nt) {
              mma_t<CT>(x[u][nt], a, qb[nt][kk][0], qb[nt][kk][1]);
              if constexpr (SPLIT) mma_t<CT>(x[u][nt], a, ql[nt][kk][0], ql[nt][kk][1]);
            }
          }
        }
        // mask + online softmax (log2 domain)
        uint32_t pb[kGroups][kNt][2], pl[SPLIT ? kGroups : 1][kNt][2];
#pragma unroll
        for (int nt = 0; nt < kNt; ++nt) {
          float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
          for (int u = 0; u < kGroups; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int tok = at[u] + g8 + (e >> 1) * 8;
              const float v = x[u][nt][e] * scale[nt][e & 1];
              x[u][nt][e] = whole || (tok >= w.lo && tok <= w.hi) ? v : -INFINITY;
              top[e & 1] = fmaxf(top[e & 1], x[u][nt][e]);
            }
          float base[2], keep[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 4));
            top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 8));
            top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 16));
            top[e] = fmaxf(top[e], m[nt][e]);
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
              l[nt][e & 1] += pr[e];
            }
            // P rounded to the pages' type: its products with V then run on
            // the tensor cores (SPLIT keeps the rest as a second operand)
            const uint32_t p0 = pack2<CT>(pr[0], pr[1]), p1 = pack2<CT>(pr[2], pr[3]);
            pb[u][nt][0] = transpose8(p0);
            pb[u][nt][1] = transpose8(p1);
            if constexpr (SPLIT) {
              pl[u][nt][0] = transpose8(pack_rest(p0, pr[0], pr[1]));
              pl[u][nt][1] = transpose8(pack_rest(p1, pr[2], pr[3]));
            }
          }
#pragma unroll
          for (int i = 0; i < D / 16; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[nt][i][e] *= keep[e & 1];
        }
        // O^T += V^T P^T: dimensions g8 and g8 + 8 of each 16
        const uint32_t vbase = smem_u32(vst);
#pragma unroll
        for (int u = 0; u < kGroups; ++u) {
          const int tok = u * 16 + vfrag_row;
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            const int chunk = 2 * i + ((lane >> 3) & 1);
            uint32_t a[4];
            ldsm_x4_t(vbase + sw128(tok * C::kHalves + (chunk >> 3), chunk & 7), a[0], a[1], a[2], a[3]);
#pragma unroll
            for (int nt = 0; nt < kNt; ++nt) {
              mma_t<CT>(o[nt][i], a, pb[u][nt][0], pb[u][nt][1]);
              if constexpr (SPLIT) mma_t<CT>(o[nt][i], a, pl[u][nt][0], pl[u][nt][1]);
            }
          }
        }
        if (!whole) fence_proxy_async_smem();  // the zeros before the next TMA into this stage
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[s]);
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
    named_barrier_sync(1, 128);
    const bool whole = sg.lt == 0 && sg.n == sg.tiles;
    float* mine = d.scratch + (static_cast<size_t>(cta) * 2 + (g == tb ? 0 : 1)) * rows * (D + 2);
    for (int i = tid; i < heads * D; i += 128) {
      const int r = i / D, c = i - r * D;
      float top = -INFINITY, sum = 0.f, v = 0.f;
#pragma unroll
      for (int k = 0; k < kConsumerWarps; ++k) top = fmaxf(top, red[(k * rows + r) * (D + 2)]);
      if (top != -INFINITY) {
#pragma unroll
        for (int k = 0; k < kConsumerWarps; ++k) {
          const float* rr = red + (k * rows + r) * (D + 2);
          const float f = ex2(rr[0] - top);
          sum += rr[1] * f;
          v += rr[2 + c] * f;
        }
      }
      if (whole) {
        store_out<IO>(d, (static_cast<int64_t>(b) * Hq + h0 + r) * D + c, sum > 0.f ? v / sum : 0.f);
      } else {
        mine[r * (D + 2) + 2 + c] = v;
        if (c == 0) {
          mine[r * (D + 2)] = top;
          mine[r * (D + 2) + 1] = sum;
        }
      }
    }
    named_barrier_sync(1, 128);  // red and q_s are free for the next segment
    g = sg.next;
  }
}

// Joins the triples of the pairs that several CTAs shared: a block per (pair,
// query head). It recomputes the shares from the positions, which it may read
// before the first kernel has finished: that kernel only starts its successor
// once its own wait for what came before is over.
constexpr int kJoinWarps = 8;
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
  float top = -INFINITY, sum = 0.f, acc[kPer];
#pragma unroll
  for (int e = 0; e < kPer; ++e) acc[e] = 0.f;
  for (int k = warp; k < n; k += kBatch * kJoinWarps) {
    float mk[kBatch], lk[kBatch], v[kBatch][kPer];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int at = k + u * kJoinWarps, slot = at < n ? slot_of[at] : -1;
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
    if (high == -INFINITY) continue;
    const float keep = ex2(top - high);
    sum *= keep;
#pragma unroll
    for (int e = 0; e < kPer; ++e) acc[e] *= keep;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const float f = ex2(mk[u] - high);
      sum += lk[u] * f;
#pragma unroll
      for (int e = 0; e < kPer; ++e) acc[e] += v[u][e] * f;
    }
    top = high;
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
  if (tid >= D) return;
  float all = 0.f, v = 0.f;
  if (high != -INFINITY) {
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) {
      const float f = ex2(red[0][w] - high);
      all += red[1][w] * f;
      v += row_s[w][tid] * f;
    }
  }
  store_out<IO>(d, static_cast<int64_t>(blockIdx.x) * D + tid, all > 0.f ? v / all : 0.f);
}

template <int D, typename CT, bool SPLIT, bool TWO>
cudaError_t launch_t(const tla_paged* P, DecodeParams& d, cudaStream_t stream) {
  using IO = typename std::conditional<SPLIT, float, CT>::type;
  auto kernel = paged_decode_kernel<D, CT, SPLIT, TWO>;
  const void* k = reinterpret_cast<const void*>(kernel);
  const int smem = smem_layout<D>(d.rows, d.p.batch, SPLIT).total;
  cudaError_t e = raise_smem_limit(k, smem);
  if (e != cudaSuccess) return e;
  // two CTAs per SM by registers (the launch bounds), if shared memory holds
  // two (228 KB, 1 KB of it reserved per CTA)
  const int per_sm = kCtasPerSm * (smem + 1024) <= 228 * 1024 ? kCtasPerSm : 1;
  const int grid = per_sm * P->base.ctx->sm_count;
  d.small_grid = P->base.ctx->sm_count;
  e = launch_pdl(kernel, grid, kThreads, smem, stream, d);
  if (e != cudaSuccess || d.whole) return e;
  return launch_pdl(paged_decode_join_kernel<D, IO>, static_cast<unsigned>(d.p.batch) * P->base.Hq, kJoinWarps * 32, 0,
                    stream, d, grid);
}

template <int D>
cudaError_t launch_d(const tla_paged* P, DecodeParams& d, cudaStream_t stream) {
  const bool two = d.rows > 8;
  if (P->io == kFp32)
    return two ? launch_t<D, __half, true, true>(P, d, stream) : launch_t<D, __half, true, false>(P, d, stream);
  if (P->kept == kBf16)
    return two ? launch_t<D, __nv_bfloat16, false, true>(P, d, stream)
               : launch_t<D, __nv_bfloat16, false, false>(P, d, stream);
  return two ? launch_t<D, __half, false, true>(P, d, stream) : launch_t<D, __half, false, false>(P, d, stream);
}

bool make_pool_map(const tla_paged* P, void* base, CUtensorMap* map) {
  const tla_page_pool& pool = P->pool;
  const cuuint64_t halves = static_cast<cuuint64_t>(P->base.D / 64);
  const int tile = P->base.D == 64 ? Cfg<64>::kTile : Cfg<128>::kTile;
  const cuuint32_t box_slots = pool.page_size < tile ? pool.page_size : tile;
  const cuuint64_t dims[5] = {64, halves, static_cast<cuuint64_t>(pool.page_size), static_cast<cuuint64_t>(P->base.Hk),
                              static_cast<cuuint64_t>(pool.page_count)};
  const cuuint64_t strides[4] = {128, static_cast<cuuint64_t>(pool.slot_stride) * 2,
                                 static_cast<cuuint64_t>(pool.head_stride) * 2,
                                 static_cast<cuuint64_t>(pool.page_stride) * 2};
  const cuuint32_t box[5] = {64, static_cast<cuuint32_t>(halves), box_slots, 1, 1};
  const cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  return P->base.ctx->encode_tiled(map,
                                   P->kept == kBf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                                   5, base, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int subgroups(const tla_paged* P) { return (P->base.G + 15) / 16; }
int subgroup_rows(const tla_paged* P) {
  const int s = subgroups(P);
  return (P->base.G + s - 1) / s;
}

}  // namespace

// The tensor-core path takes 16-bit pages of 16 tokens and up (a warp's 16
// tokens lie in one page), head_dim 64 or 128 and pools that a tensor map can
// describe; float32 activations only over float16 pages (two bfloat16 parts
// would carry 16 bits).
void paged_decode_configure(tla_paged* P) {
  const tla_page_pool& pool = P->pool;
  P->fast = false;
  if (!P->wide || P->kept == kFp32 || (P->io == kFp32 && P->kept != kFp16) || pool.page_size < 16 || P->base.ctx->encode_tiled == nullptr ||
      kCtasPerSm * P->base.ctx->sm_count > kMaxGrid)
    return;
  tla_paged q = *P;
  if (pool.page_count == 1) q.pool.page_stride = P->base.D;
  if (P->base.Hk == 1) q.pool.head_stride = P->base.D;
  P->fast = make_pool_map(&q, pool.key, &P->tmap_k) && make_pool_map(&q, pool.value, &P->tmap_v);
}

// The most tiles that a pair of this call can have.
long long most_tiles(const PagedArgs& p, int count) {
  const int kTile = p.a.D == 64 ? Cfg<64>::kTile : Cfg<128>::kTile;
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

#ifndef WHOLE
#define WHOLE 20
#endif
bool whole_pairs(const PagedArgs& p, int count) { return most_tiles(p, count) <= WHOLE; }

// Whether a call's shares can be cut: the batch's table fits shared memory and
// its tiles are counted in 32 bits.
bool paged_decode_takes(const tla_paged* P, const PagedArgs& p, int count) {
  return P->fast && p.batch <= kMaxBatch &&
         (most_tiles(p, count) + 16) * p.a.Hk * subgroups(P) * p.batch < (1LL << 31);
}

size_t paged_decode_workspace(const tla_paged* P, const PagedArgs& p, int count) {
  if (whole_pairs(p, count)) return 0;
  return static_cast<size_t>(kCtasPerSm) * P->base.ctx->sm_count * 2 * subgroup_rows(P) * (P->base.D + 2) *
         sizeof(float);
}

cudaError_t launch_paged_decode(const tla_paged* P, const PagedArgs& p, const void* query, const int32_t* pages,
                                int count, const void* gate, void* out, void* workspace, cudaStream_t stream) {
  DecodeParams d;
  d.tmap_k = P->tmap_k;
  d.tmap_v = P->tmap_v;
  d.p = p;
  d.query = query;
  d.pages = pages;
  d.gate = gate;
  d.out = out;
  d.scratch = static_cast<float*>(workspace);
  d.count = count;
  d.subs = subgroups(P);
  d.rows = subgroup_rows(P);
  d.small_grid = 0;
  d.whole = whole_pairs(p, count) ? 1 : 0;
  return P->base.D == 64 ? launch_d<64>(P, d, stream) : launch_d<128>(P, d, stream);
}

}  // namespace tla
