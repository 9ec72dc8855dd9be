// C ABI of the paged key-value cache: layers over a caller's page pool,
// argument checks and dispatch. No entry point allocates after
// tla_paged_create or keeps anything between calls.
#include <math.h>

#include <memory>
#include <new>
#include <utility>

#include "tla_device.cuh"
#include "tla_host.h"
#include "tla_internal.h"

namespace tla {

PagedArgs paged_args(const tla_paged* P, const int32_t* positions, const int32_t* table, int width, int batch) {
  PagedArgs p;
  p.a = layer_args(&P->base);
  p.key = P->pool.key;
  p.value = P->pool.value;
  p.bounds = P->pool.bounds;
  p.page_stride = P->pool.page_stride;
  p.head_stride = P->pool.head_stride;
  p.slot_stride = P->pool.slot_stride;
  p.table = table;
  p.positions = positions;
  p.turns = P->d_turns;
  p.width = width;
  p.batch = batch;
  p.page_count = P->pool.page_count;
  p.page_shift = P->page_shift;
  const long long held = static_cast<long long>(width) << P->page_shift;
  p.capacity = static_cast<int>(held < P->base.max_tokens ? held : P->base.max_tokens);
  return p;
}

}  // namespace tla

using tla::DeviceGuard;
using tla::from_cuda;

namespace {

// The call's common arguments; TLA_OK when there is work to do or batch is 0.
int check_call(const tla_paged* P, const void* positions, const void* table, int32_t width, int32_t batch) {
  if (!P || batch < 0 || batch > P->base.max_batch || width <= 0) return TLA_ERR_INVALID_ARG;
  if (batch > 0 && (!positions || !table)) return TLA_ERR_INVALID_ARG;
  return TLA_OK;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Whether rows of activations may start there: on 16 bytes where head_dim is a
// multiple of 8 (the kernels then read and write several elements at a time;
// every row of a dense tensor does), else on an element.
bool row_start(const tla_paged* P, const void* p) {
  const int step = P->base.D % 8 == 0 ? 16 : P->io == tla::kFp32 ? 4 : 2;
  return reinterpret_cast<uintptr_t>(p) % step == 0;
}

// Whether every (page, head, slot) row of D elements has memory of its own:
// sorted by stride, each dimension must step over all that the smaller span.
bool rows_apart(const tla_page_pool& pool, int heads, int D) {
  std::pair<int64_t, int64_t> dim[3] = {
      {pool.page_stride, pool.page_count}, {pool.head_stride, heads}, {pool.slot_stride, pool.page_size}};
  for (int i = 0; i < 2; ++i)
    for (int j = 0; j < 2 - i; ++j)
      if (dim[j + 1].first < dim[j].first) std::swap(dim[j], dim[j + 1]);
  int64_t span = D;
  for (const auto& d : dim) {
    if (d.second == 1) continue;
    if (d.first < span || d.first > (int64_t(1) << 40)) return false;
    span = d.first * (d.second - 1) + span;
  }
  return true;
}

// Whether [a, a + n) and [b, b + m) share a byte.
bool overlap(const void* a, size_t n, const void* b, size_t m) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return a && b && x < y + m && y < x + n;
}
size_t row_bytes(const tla_paged* P, int heads) {
  return static_cast<size_t>(heads) * P->base.D * (P->io == tla::kFp32 ? 4 : 2);
}

size_t decode_workspace(const tla_paged* P, const tla::PagedArgs& p, int count) {
  return tla::paged_decode_takes(P, p, count) ? tla::paged_decode_workspace(P, p, count)
                                              : tla::paged_decode_generic_workspace(P, p.batch);
}

}  // namespace

extern "C" {

int tla_paged_create(tla_ctx* ctx, const tla_attn_config* cfg, const tla_page_pool* pool, const float* q_norm_weight,
                     const float* k_norm_weight, tla_paged** out) try {
  if (!out) return TLA_ERR_INVALID_ARG;
  *out = nullptr;
  if (!ctx || !cfg || !pool || !pool->key || !pool->value || pool->key == pool->value) return TLA_ERR_INVALID_ARG;
  tla_layer L;
  std::vector<float> inv;
  int rc = tla::layer_params(cfg, &L, &inv);
  if (rc != TLA_OK) return rc;
  // query heads that do not divide into the kv heads; more heads than a grid's second dimension
  if (L.G == 0 || L.Hq > 65535) return TLA_ERR_UNSUPPORTED;
  const uint32_t io_bits = cfg->flags & (TLA_FLAG_IO_FP32 | TLA_FLAG_IO_BF16);
  const uint32_t kept_bits = cfg->flags & (TLA_FLAG_CACHE_FP32 | TLA_FLAG_CACHE_BF16);
  if (io_bits == (TLA_FLAG_IO_FP32 | TLA_FLAG_IO_BF16) || kept_bits == (TLA_FLAG_CACHE_FP32 | TLA_FLAG_CACHE_BF16))
    return TLA_ERR_INVALID_ARG;
  const int io = io_bits == TLA_FLAG_IO_FP32 ? tla::kFp32 : io_bits == TLA_FLAG_IO_BF16 ? tla::kBf16 : tla::kFp16;
  const int kept = kept_bits == TLA_FLAG_CACHE_FP32 ? tla::kFp32
                   : kept_bits == TLA_FLAG_CACHE_BF16 ? tla::kBf16 : tla::kFp16;
  if (io != kept && io != tla::kFp32) return TLA_ERR_UNSUPPORTED;
  if (pool->page_count <= 0 || pool->page_size <= 0 || pool->page_size > 1024 ||
      (pool->page_size & (pool->page_size - 1)) != 0)
    return TLA_ERR_INVALID_ARG;
  if (!rows_apart(*pool, L.Hk, L.D)) return TLA_ERR_INVALID_ARG;
  const size_t elem = kept == tla::kFp32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(pool->key) % elem || reinterpret_cast<uintptr_t>(pool->value) % elem ||
      !aligned16(pool->bounds))
    return TLA_ERR_INVALID_ARG;
  DeviceGuard g(ctx->device);
  std::unique_ptr<tla_paged, int (*)(tla_paged*)> owner(new tla_paged(), tla_paged_destroy);
  tla_paged* P = owner.get();
  P->base.ctx = ctx;
  L.ctx = ctx;
  L.k_cache = pool->key;
  L.v_cache = pool->value;
  L.borrowed = true;  // the pool is the caller's
  P->base = L;
  P->pool = *pool;
  P->io = io;
  P->kept = kept;
  while ((1 << P->page_shift) < pool->page_size) ++P->page_shift;
  // a dimension of one entry may carry any stride
  const int vec = static_cast<int>(16 / elem);
  P->wide = L.D % 8 == 0 && aligned16(pool->key) && aligned16(pool->value) &&
            (pool->page_count == 1 || pool->page_stride % vec == 0) && (L.Hk == 1 || pool->head_stride % vec == 0) &&
            (pool->page_size == 1 || pool->slot_stride % vec == 0);
  rc = from_cuda(tla::paged_decode_configure(P));
  if (rc == TLA_OK) rc = tla::layer_tables(&P->base, inv, q_norm_weight, k_norm_weight);
  const int half = L.rotary / 2;
  if (rc == TLA_OK && half > 0) {
    std::vector<float2> turns(static_cast<size_t>(tla::kTurnSteps) * half);
    for (int s = 0; s < tla::kTurnSteps; ++s)
      for (int j = 0; j < half; ++j) {
        const double angle = j < L.pair_count ? s * static_cast<double>(inv[j]) : 0.0;
        turns[static_cast<size_t>(s) * half + j] =
            make_float2(static_cast<float>(cos(angle)), static_cast<float>(sin(angle)));
      }
    rc = tla::dev_alloc(&P->d_turns, turns.size());
    if (rc == TLA_OK)
      rc = from_cuda(cudaMemcpy(P->d_turns, turns.data(), turns.size() * sizeof(float2), cudaMemcpyHostToDevice));
  }
  if (rc != TLA_OK) return rc;
  *out = owner.release();
  return TLA_OK;
} catch (const std::bad_alloc&) {
  return TLA_ERR_OUT_OF_MEMORY;
} catch (...) {
  return TLA_ERR_INVALID_ARG;
}

int tla_paged_destroy(tla_paged* P) {
  if (!P) return TLA_OK;
  DeviceGuard g(P->base.ctx->device);
  cudaFree(P->d_turns);
  cudaFree(P->base.d_inv_freq);
  cudaFree(P->base.d_qnorm);
  cudaFree(P->base.d_knorm);
  delete P;
  return TLA_OK;
}

int tla_paged_append(tla_paged* P, const void* qkv, const int32_t* positions, const int32_t* row_offsets,
                     const int32_t* page_table, int32_t table_width, int32_t batch, int32_t rows, void* query_out,
                     void* stream) {
  int rc = check_call(P, positions, page_table, table_width, batch);
  if (rc != TLA_OK) return rc;
  if (rows < 0 || (rows > 0 && !qkv) || (!row_offsets && rows != batch)) return TLA_ERR_INVALID_ARG;
  if (batch == 0 || rows == 0) return TLA_OK;
  if (!row_start(P, qkv) || !row_start(P, query_out) ||
      overlap(qkv, rows * row_bytes(P, P->base.Hq + 2 * P->base.Hk), query_out, rows * row_bytes(P, P->base.Hq)))
    return TLA_ERR_INVALID_ARG;
  if (!tla::paged_append_takes(P)) return TLA_ERR_UNSUPPORTED;
  DeviceGuard g(P->base.ctx->device);
  return from_cuda(tla::launch_paged_append(P, tla::paged_args(P, positions, page_table, table_width, batch), qkv,
                                            row_offsets, rows, query_out, static_cast<cudaStream_t>(stream)));
}

int tla_paged_workspace(const tla_paged* P, int32_t batch, int32_t table_width, int32_t page_count,
                        size_t* decode_bytes, size_t* select_bytes) {
  if (!P || batch < 0 || batch > P->base.max_batch || table_width <= 0 || page_count < 0) return TLA_ERR_INVALID_ARG;
  const tla::PagedArgs p = tla::paged_args(P, nullptr, nullptr, table_width, batch);
  if (decode_bytes) *decode_bytes = batch > 0 ? decode_workspace(P, p, page_count) : 0;
  if (select_bytes) *select_bytes = tla::paged_select_workspace(P, batch, table_width);
  return TLA_OK;
}

int tla_paged_decode(tla_paged* P, const void* query, const int32_t* positions, const int32_t* page_table,
                     int32_t table_width, const int32_t* pages, int32_t page_count, const void* gate, void* out,
                     int32_t batch, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_call(P, positions, page_table, table_width, batch);
  if (rc != TLA_OK) return rc;
  if (batch == 0) return page_count < 0 ? TLA_ERR_INVALID_ARG : TLA_OK;  // (an empty list's address may be null)
  if (pages ? page_count <= 0 : page_count != 0) return TLA_ERR_INVALID_ARG;
  const size_t bytes = batch * row_bytes(P, P->base.Hq);
  if (!query || !out || !row_start(P, query) || !row_start(P, out) || !row_start(P, gate) || !aligned16(workspace) ||
      overlap(query, bytes, out, bytes) || (gate != out && overlap(gate, bytes, out, bytes)))
    return TLA_ERR_INVALID_ARG;
  const tla::PagedArgs p = tla::paged_args(P, positions, page_table, table_width, batch);
  const size_t need = decode_workspace(P, p, page_count);
  if (need > 0 && (!workspace || workspace_bytes < need)) return TLA_ERR_INVALID_ARG;
  DeviceGuard g(P->base.ctx->device);
  if (tla::paged_decode_takes(P, p, page_count))
    return from_cuda(tla::launch_paged_decode(P, p, query, pages, page_count, gate, out, workspace,
                                              static_cast<cudaStream_t>(stream)));
  return from_cuda(tla::launch_paged_decode_generic(P, p, query, pages, page_count, gate, out, workspace,
                                                    static_cast<cudaStream_t>(stream)));
}

int tla_paged_select(tla_paged* P, const void* query, const int32_t* positions, const int32_t* page_table,
                     int32_t table_width, int32_t first_pages, int32_t last_pages, int32_t* pages_out,
                     int32_t page_count, int32_t batch, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_call(P, positions, page_table, table_width, batch);
  if (rc != TLA_OK) return rc;
  if (page_count <= 0 || first_pages < 0 || last_pages < 0 ||
      static_cast<int64_t>(first_pages) + last_pages > page_count)
    return TLA_ERR_INVALID_ARG;
  if (!P->pool.bounds || !(P->base.attn_scale > 0)) return TLA_ERR_UNSUPPORTED;
  if (batch == 0) return TLA_OK;
  if (!query || !pages_out || !row_start(P, query) || !aligned16(workspace) ||
      overlap(query, batch * row_bytes(P, P->base.Hq), pages_out,
              static_cast<size_t>(batch) * P->base.Hk * page_count * sizeof(int32_t)))
    return TLA_ERR_INVALID_ARG;
  const size_t need = tla::paged_select_workspace(P, batch, table_width);
  if (need > 0 && (!workspace || workspace_bytes < need)) return TLA_ERR_INVALID_ARG;
  DeviceGuard g(P->base.ctx->device);
  const tla::PagedArgs p = tla::paged_args(P, positions, page_table, table_width, batch);
  return from_cuda(tla::launch_paged_select(P, p, query, first_pages, last_pages, pages_out, page_count, workspace,
                                            static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
