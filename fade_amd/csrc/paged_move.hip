// Tokens moved within the pages of a cache, in K and V of every layer by one launch.
//
// fade_paged_copy: the first tokens of a page to a page of its own (what page_fork lists).
// A workgroup takes one copy in one tensor and kv head: [tokens][D] is one run of bytes on
// both sides.
//
// fade_paged_compact: of a row's drafted tokens those on the accepted path to the first
// places of them.  Numbers on a path rise, path[i] >= i, so a token moves to its own place
// or an earlier one; a thread takes 16 bytes of a head's channels down the whole path, eight
// tokens read before the eight are written: what later ones read lies behind that.  No
// thread touches another's bytes, so nothing waits.
// Both bound by HBM where much is moved, else by latency (counts, table, page): the partial pages
// of 96 beams in 16 layers (154 MB read and written, in part from the last-level cache) 23.5 us,
// four samples' in 24 small layers 3.3; the accepted ones of 64 rows' 24 tokens in 28 layers (19 MB) 8.2, of 64 tokens in layers of
// eight heads (68 MB) 15.5, of one row 3.8.
#include "fade_common.h"

namespace fade {
namespace move {
namespace {

constexpr int kPage = 64;
constexpr int kThreads = 256;
constexpr int kPools = 128;  // tensors of a launch

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct Pools {
  u32x4* at[kPools];
};

struct CopyParams {
  const int32_t* copies;
  int64_t n_pages;
  int Hkv, units;  // 16-byte units of a token in a head
};

__global__ __launch_bounds__(kThreads) void copy_kernel(Pools pools, CopyParams p) {
  const int r = blockIdx.x / p.Hkv, h = blockIdx.x - r * p.Hkv;
  const int64_t src = p.copies[3 * r], dst = p.copies[3 * r + 1];
  int n = p.copies[3 * r + 2];
  if (src < 1 || src >= p.n_pages || dst < 1 || dst >= p.n_pages || n < 1) return;
  n = (n > kPage ? kPage : n) * p.units;
  const u32x4* const from = pools.at[blockIdx.y] + (src * p.Hkv + h) * kPage * p.units;
  u32x4* const to = pools.at[blockIdx.y] + (dst * p.Hkv + h) * kPage * p.units;
  constexpr int K = 4;
  for (int i = threadIdx.x; i < n; i += K * kThreads) {
    u32x4 x[K];
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (i + k * kThreads < n) x[k] = from[i + k * kThreads];
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (i + k * kThreads < n) to[i + k * kThreads] = x[k];
  }
}

struct CompactParams {
  int64_t max_path, ppr, n_pages;
  int Hkv, units, slices;  // slices of a token's units over workgroups
  const int32_t* path;
  const int32_t* counts;
  const int32_t* table;
  const int32_t* lens;
  const int32_t* starts;
  int32_t* kept;  // or null
};

__global__ __launch_bounds__(kThreads) void compact_kernel(Pools pools, CompactParams p) {
  constexpr int kMoves = 256;  // at once
  __shared__ int64_t from[kMoves], to[kMoves];  // the token's first unit in head 0; -1: no move
  const int b = blockIdx.x / p.slices, slice = blockIdx.x - b * p.slices;
  int n = p.starts[b + 1] - p.starts[b];
  n = n < 0 ? 0 : n;
  const int len = p.lens[b] < 0 ? 0 : p.lens[b], base = len - n, cap = static_cast<int>(p.ppr) * kPage;
  int count = p.counts[b];
  count = count < 0 ? 0 : (count > n ? n : count);
  count = count > p.max_path ? static_cast<int>(p.max_path) : count;
  if (p.kept != nullptr && blockIdx.y == 0 && slice == 0 && threadIdx.x == 0) p.kept[b] = base + count < 0 ? 0 : base + count;
  if (base < 0 || len > cap) return;
  const int columns = p.Hkv * p.units;
  const int32_t* const trow = p.table + b * p.ppr;
  for (int m0 = 0; m0 < count; m0 += kMoves) {
    const int m = count - m0 < kMoves ? count - m0 : kMoves;
    __syncthreads();
    for (int i = threadIdx.x; i < m; i += kThreads) {
      const int x = p.path[b * p.max_path + m0 + i];
      int64_t f = -1, t = -1;
      if (x >= 0 && x < n && x != m0 + i) {
        const int a = base + x, c = base + m0 + i;
        const int64_t pa = trow[a / kPage], pc = trow[c / kPage];
        if (pa >= 1 && pa < p.n_pages && pc >= 1 && pc < p.n_pages) {
          f = (pa * p.Hkv * kPage + a % kPage) * p.units;
          t = (pc * p.Hkv * kPage + c % kPage) * p.units;
        }
      }
      from[i] = f;
      to[i] = t;
    }
    __syncthreads();
    for (int col = slice * kThreads + threadIdx.x; col < columns; col += p.slices * kThreads) {
      const int h = col / p.units;
      u32x4* const at = pools.at[blockIdx.y] + static_cast<int64_t>(h) * kPage * p.units + (col - h * p.units);
      constexpr int K = 8;
      for (int i = 0; i < m; i += K) {
        u32x4 x[K];
#pragma unroll
        for (int k = 0; k < K; ++k)
          if (i + k < m && from[i + k] >= 0) x[k] = at[from[i + k]];
#pragma unroll
        for (int k = 0; k < K; ++k)
          if (i + k < m && from[i + k] >= 0) at[to[i + k]] = x[k];
      }
    }
  }
}

int check_args(const fade_paged_move_args* a, const char* what) {
  if (a == nullptr) return einval("%s: null args", what);
  if (a->n_pools < 1 || a->n_pools > 65535 || a->n_pages < 1 || a->n_pages >= (1ll << 31) || a->Hkv < 1 || a->Hkv > 65535)
    return einval("%s: n_pools and Hkv must be 1 to 65535, n_pages 1 to 2^31 - 1", what);
  if (a->D < 8 || a->D > 256 || a->D % 8) return einval("%s: head_dim must be a multiple of 8 in [8, 256], got %lld", what, (long long)a->D);
  if (a->rows < 0 || a->rows > (1 << 20)) return einval("%s: too many rows", what);
  if (!a->pools) return einval("%s: null pools", what);
  for (int64_t i = 0; i < a->n_pools; ++i)
    if (!a->pools[i] || (reinterpret_cast<uintptr_t>(a->pools[i]) & 15)) return einval("%s: pools must be 16-byte aligned", what);
  return FADE_OK;
}

// launch(tensors, how many, number of the first, rows r0 .., how many of them), `per_row` workgroups a row; a launch
// has fewer than 2^32 threads along x.
template <class F>
int each_launch(const fade_paged_move_args* a, int64_t per_row, const char* what, F&& launch) {
  const int64_t most = ((1ll << 32) / kThreads - 1) / per_row;
  for (int64_t i0 = 0; i0 < a->n_pools; i0 += kPools) {
    Pools pools;
    const int64_t n = a->n_pools - i0 < kPools ? a->n_pools - i0 : kPools;
    for (int64_t i = 0; i < n; ++i) pools.at[i] = static_cast<u32x4*>(a->pools[i0 + i]);
    for (int64_t r0 = 0; r0 < a->rows; r0 += most) {
      launch(pools, static_cast<unsigned>(n), i0, r0, a->rows - r0 < most ? a->rows - r0 : most);
      const int rc = check_launch(what);
      if (rc) return rc;
    }
  }
  return FADE_OK;
}

}  // namespace
}  // namespace move
}  // namespace fade

using namespace fade;
using namespace fade::move;

FADE_API int fade_paged_copy(const fade_paged_move_args* a, void* stream) {
  const char* what = "fade_paged_copy";
  const int rc = check_args(a, what);
  if (rc) return rc;
  if (a->rows == 0) return FADE_OK;
  if (!a->copies) return einval("%s: null copies", what);
  return each_launch(a, a->Hkv, what, [&](const Pools& pools, unsigned n, int64_t, int64_t r0, int64_t rows) {
    const CopyParams p{a->copies + 3 * r0, a->n_pages, static_cast<int>(a->Hkv), static_cast<int>(a->D / 8)};
    hipLaunchKernelGGL(copy_kernel, dim3(static_cast<unsigned>(rows * a->Hkv), n), dim3(kThreads), 0, as_stream(stream), pools, p);
  });
}

FADE_API int fade_paged_compact(const fade_paged_move_args* a, void* stream) {
  const char* what = "fade_paged_compact";
  const int rc = check_args(a, what);
  if (rc) return rc;
  if (a->max_path < 1 || a->max_path > FADE_DRAFT_MAX_NODES || a->pages_per_row < 1 || a->pages_per_row > (1 << 24))
    return einval("%s: max_path must be 1 to %d, pages_per_row 1 to 2^24", what, FADE_DRAFT_MAX_NODES);
  if (a->rows < 1 || !a->path || !a->counts || !a->table || !a->lens || !a->starts || !a->kept)
    return einval("%s: needs rows, path, counts, table, lens, starts and kept", what);
  const int64_t slices = cdiv(a->Hkv * (a->D / 8), kThreads);
  return each_launch(a, slices, what, [&](const Pools& pools, unsigned n, int64_t i0, int64_t r0, int64_t rows) {
    CompactParams p;
    p.max_path = a->max_path;
    p.ppr = a->pages_per_row;
    p.n_pages = a->n_pages;
    p.Hkv = static_cast<int>(a->Hkv);
    p.units = static_cast<int>(a->D / 8);
    p.slices = static_cast<int>(slices);
    p.path = a->path + r0 * a->max_path;
    p.counts = a->counts + r0;
    p.table = a->table + r0 * a->pages_per_row;
    p.lens = a->lens + r0;
    p.starts = a->starts + r0;
    p.kept = i0 == 0 ? a->kept + r0 : nullptr;
    hipLaunchKernelGGL(compact_kernel, dim3(static_cast<unsigned>(rows * slices), n), dim3(kThreads), 0, as_stream(stream), pools, p);
  });
}
