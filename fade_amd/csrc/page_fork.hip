// Rows of a paged cache that go on from other rows: samples of one prompt, beams, rows
// shortened to the drafted tokens that were accepted, rows dropped.
//
// Row r of the result holds the first n_r tokens of row source[r], in the same pages.  A
// page may so have several holders; what a row writes next goes into its last page, where
// that is not full, so that page has to be its own.  With
//   h(P) = rows of the result that hold page P, e(P) = rows that end in it (not full),
// row r that ends in P keeps it where h(P) = e(P) and no row before r ends in it, and gets a
// copy on a free page otherwise.  Pages that were held and for which h(P) = 0 go behind the
// ring's tail by number.  Which page goes where follows from sums over rows and over pages,
// never from the order in which workgroups run.
//
// Holders are counted anew at each call, from the tables: nothing has to be kept between
// calls that could come apart from them.
//
// Large calls take four launches, as a sum over all rows has to be whole before the next
// step: words cleared, rows counted, pages without a holder counted by segments, all written.
// Each is bound by latency (1000 rows of 64 entries over 18000 pages 22 us, 64 of 512 15 us).
#include "fade_common.h"

namespace fade {
namespace fork {
namespace {

constexpr int kPage = 64;
constexpr int kThreads = 256;
constexpr int kSegment = 1024;          // pages
constexpr uint32_t kHeld = 1u << 31;    // a page's word: held before, rows that end in it, rows that hold it
constexpr uint32_t kEnds = 1u << 13;
constexpr uint32_t kCount = kEnds - 1;  // (4096 rows at most)

struct Params {
  int B, R, ppr, cap;
  const int32_t* lens;
  const int32_t* source;
  const int32_t* keep;
  const int32_t* table;
  int32_t* free_pages;
  const int32_t* ring;
  const int32_t* before;  // status of an earlier call, or null
  int32_t* table_out;
  int32_t* lens_out;
  int32_t* copies;
  int32_t* ring_out;
  int32_t* status;
  uint32_t* word;    // [cap + 1]
  uint32_t* first;   // [cap + 1]: R less the first row that ends in the page
  uint32_t* left;    // [segments]: pages without a holder
  uint32_t* bad;     // [2]: impossible counts; all pages without a holder
};

__device__ __forceinline__ int pages_of(int tokens) { return (tokens + (kPage - 1)) / kPage; }

// Row r's source and tokens; false where they cannot be.
__device__ __forceinline__ bool row_of(const Params& p, int r, int& src, int& n) {
  src = p.source != nullptr ? p.source[r] : r;
  n = 0;
  if (src < -1 || src >= p.B) return false;
  const int keep = p.keep != nullptr ? p.keep[r] : 0x7FFFFFFF;
  if (src >= 0) {
    const int len = p.lens[src];
    if (len < 0 || len > static_cast<int64_t>(p.ppr) * kPage) return false;
    n = len < keep ? len : keep;
  }
  return keep >= 0;
}

__global__ __launch_bounds__(kThreads) void fork_clear_kernel(uint32_t* at, int64_t n) {
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * kThreads) at[i] = 0;
}

// The status bits of an earlier call that was not done.
__device__ __forceinline__ int failed_before(const Params& p) {
  const int x = p.before != nullptr ? p.before[0] : 0;
  return ((x | x >> 8) & 0xFF) << 8;
}

// The words of all pages.
__global__ __launch_bounds__(kThreads) void fork_count_kernel(Params p) {
  const int spans = (p.ppr + kThreads - 1) / kThreads;
  for (int64_t item = blockIdx.x; item < static_cast<int64_t>(p.B + p.R) * spans; item += gridDim.x) {
    const int row = static_cast<int>(item / spans), j = static_cast<int>(item - static_cast<int64_t>(row) * spans) * kThreads + threadIdx.x;
    bool ok = true;
    int src = row, n = 0;
    if (row < p.B) {
      n = p.lens[row];
      ok = n >= 0 && n <= static_cast<int64_t>(p.ppr) * kPage;
    } else {
      ok = row_of(p, row - p.B, src, n);
    }
    if (ok && j < pages_of(n)) {
      const int id = p.table[static_cast<int64_t>(src) * p.ppr + j];
      if (id < 1 || id > p.cap) {
        ok = false;
      } else if (row < p.B) {
        atomicOr(&p.word[id], kHeld);
      } else {
        const bool end = (j + 1) * static_cast<int64_t>(kPage) > n;
        atomicAdd(&p.word[id], end ? kEnds + 1 : 1u);
        if (end) atomicMax(&p.first[id], static_cast<uint32_t>(p.R - (row - p.B)));
      }
    }
    if (!ok) atomicOr(p.bad, 1u);
  }
}

__device__ __forceinline__ bool is_left(uint32_t w) { return (w & kHeld) != 0 && (w & kCount) == 0; }

__global__ __launch_bounds__(kThreads) void fork_left_kernel(Params p) {
  __shared__ uint32_t sum;
  if (threadIdx.x == 0) sum = 0;
  __syncthreads();
  uint32_t n = 0;
  for (int i = threadIdx.x; i < kSegment; i += kThreads) {
    const int64_t id = static_cast<int64_t>(blockIdx.x) * kSegment + i;
    if (id >= 1 && id <= p.cap && is_left(p.word[id])) ++n;
  }
  if (n) atomicAdd(&sum, n);
  __syncthreads();
  if (threadIdx.x == 0) {
    p.left[blockIdx.x] = sum;
    if (sum) atomicAdd(&p.bad[1], sum);
  }
}

// Exclusive sum over the workgroup's threads; all: of all of them.
template <int THREADS>
__device__ __forceinline__ int block_scan(int v, int32_t* s_wave, int& all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int it = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int x = __shfl_up(it, o, 64);
    if (lane >= o) it += x;
  }
  __syncthreads();
  if (lane == 63) s_wave[wave] = it;
  __syncthreads();
  all = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) {
    if (w < wave) it += s_wave[w];
    all += s_wave[w];
  }
  return it - v;
}

template <int ROWS>
__global__ __launch_bounds__(kThreads) void fork_write_kernel(Params p) {
  constexpr int PER = ROWS / kThreads;
  __shared__ int32_t s_src[ROWS], s_n[ROWS], s_copy[ROWS];  // the row's number among the copies, or -1
  __shared__ int32_t s_wave[kThreads / 64];
  const int tid = threadIdx.x;
  const int head = p.ring[0], count = p.ring[1], left = static_cast<int>(p.bad[1]);
  int fail = (p.bad[0] ? FADE_SLOTS_BAD_COUNT : 0) | failed_before(p);
  int mine = 0;
  uint32_t flags = 0;
  if (!fail) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int r = tid * PER + i;
      if (r >= p.R) continue;
      int src, n;
      row_of(p, r, src, n);
      s_src[r] = src;
      s_n[r] = n;
      if (n % kPage == 0) continue;
      const int id = p.table[static_cast<int64_t>(src) * p.ppr + n / kPage];
      const uint32_t w = p.word[id];
      if ((w & kCount) == ((w & ~kHeld) / kEnds) && static_cast<int>(p.first[id]) == p.R - r) continue;
      flags |= 1u << i;
      ++mine;
    }
  }
  int copies;
  int at = block_scan<kThreads>(mine, s_wave, copies);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int r = tid * PER + i;
    if (r < p.R) s_copy[r] = (flags >> i & 1u) ? at++ : -1;
  }
  if (head < 0 || head >= p.cap || count < 0 || count > p.cap - left) fail |= FADE_SLOTS_BAD_COUNT;
  else if (copies > count) fail |= FADE_SLOTS_EXHAUSTED;
  __syncthreads();

  const int64_t stride = static_cast<int64_t>(gridDim.x) * kThreads, first = static_cast<int64_t>(blockIdx.x) * kThreads + tid;
  if (fail) {  // nothing changes
    for (int64_t e = first; e < static_cast<int64_t>(p.R) * p.ppr; e += stride) p.table_out[e] = e / p.ppr < p.B ? p.table[e] : 0;
    for (int64_t r = first; r < p.R; r += stride) {
      p.lens_out[r] = r < p.B ? p.lens[r] : 0;
      p.copies[3 * r] = p.copies[3 * r + 1] = p.copies[3 * r + 2] = 0;
    }
    if (first == 0) {
      p.ring_out[0] = head;
      p.ring_out[1] = count;
      p.status[0] = fail;
    }
    return;
  }
  const uint32_t cap = static_cast<uint32_t>(p.cap);
  auto taken = [&](int i) { return p.free_pages[(static_cast<uint32_t>(head) + static_cast<uint32_t>(i)) % cap]; };
  const int spans = (p.ppr + kThreads - 1) / kThreads;
  for (int64_t item = blockIdx.x; item < static_cast<int64_t>(p.R) * spans; item += gridDim.x) {
    const int r = static_cast<int>(item / spans), j = static_cast<int>(item - static_cast<int64_t>(r) * spans) * kThreads + tid;
    if (j >= p.ppr) continue;
    const int pages = pages_of(s_n[r]);
    int id = 0;
    if (j < pages) id = j == pages - 1 && s_copy[r] >= 0 ? taken(s_copy[r]) : p.table[static_cast<int64_t>(s_src[r]) * p.ppr + j];
    p.table_out[static_cast<int64_t>(r) * p.ppr + j] = id;
  }
  for (int64_t r = first; r < p.R; r += stride) {
    const int n = s_n[r], c = s_copy[r];
    p.lens_out[r] = n;
    p.copies[3 * r] = c < 0 ? 0 : p.table[static_cast<int64_t>(s_src[r]) * p.ppr + n / kPage];
    p.copies[3 * r + 1] = c < 0 ? 0 : taken(c);
    p.copies[3 * r + 2] = c < 0 ? 0 : n % kPage;
  }
  if (first == 0) {
    p.ring_out[0] = static_cast<int32_t>((static_cast<uint32_t>(head) + static_cast<uint32_t>(copies)) % cap);
    p.ring_out[1] = count - copies + left;
    p.status[0] = 0;
  }
  // the pages without a holder, a segment after the other
  const int segments = p.cap / kSegment + 1;
  for (int g = blockIdx.x; g < segments; g += gridDim.x) {
    if (p.left[g] == 0) continue;
    int ahead = 0, all;
    for (int i = tid; i < g; i += kThreads) ahead += static_cast<int>(p.left[i]);
    block_scan<kThreads>(ahead, s_wave, all);
    ahead = all;
    constexpr int EACH = kSegment / kThreads;
    uint32_t mask = 0;
    int n = 0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int64_t id = static_cast<int64_t>(g) * kSegment + tid * EACH + i;
      if (id >= 1 && id <= p.cap && is_left(p.word[id])) {
        mask |= 1u << i;
        ++n;
      }
    }
    int to = ahead + block_scan<kThreads>(n, s_wave, all);
#pragma unroll
    for (int i = 0; i < EACH; ++i)
      if (mask >> i & 1u) p.free_pages[(static_cast<uint64_t>(head) + count + to++) % cap] = g * kSegment + tid * EACH + i;
  }
}

// Small calls: all of it in one workgroup, the pages' words in LDS.  Bound by latency: counts, table (twice), the
// written entries.  On the GPU, and a call: 4 rows of 16 entries 5.2 us and 12.3, by the four launches above
// 10.8 and 21.6; 16 of 64 6.0 / 12.6, 13.4 / 21.2; 64 of 128 13.2 / 12.9, 14.8 / 21.3; past that the workgroup's
// walk over the tables is what counts (64 of 512 33, 15 by the launches).
constexpr int kSmallThreads = 1024;
constexpr int kSmallRows = kSmallThreads;  // one a thread
constexpr int kSmallPages = 16384;
constexpr int kSmallEntries = 16384;  // of both tables

__global__ __launch_bounds__(kSmallThreads) void fork_small_kernel(Params p) {
  __shared__ uint32_t word[kSmallPages + 1], begun[kSmallPages + 1];
  __shared__ int32_t s_len[kSmallRows], s_src[kSmallRows], s_n[kSmallRows], s_copy[kSmallRows];
  __shared__ int32_t s_wave[kSmallThreads / 64];
  __shared__ uint32_t s_bad;
  const int tid = threadIdx.x, ppr = p.ppr;
  const int head = p.ring[0], count = p.ring[1], before = failed_before(p);
  int len = tid < p.B ? p.lens[tid] : 0;
  int src = tid >= p.R ? -1 : (p.source != nullptr ? p.source[tid] : tid);
  const int keep = p.keep != nullptr && tid < p.R ? p.keep[tid] : 0x7FFFFFFF;
  if (tid == 0) s_bad = 0;
  for (int i = tid; i <= p.cap; i += kSmallThreads) word[i] = begun[i] = 0;
  bool ok = len >= 0 && len <= static_cast<int64_t>(ppr) * kPage && src >= -1 && src < p.B && keep >= 0;
  if (!ok) {
    len = 0;
    src = -1;
  }
  s_len[tid] = len;
  s_src[tid] = src;
  __syncthreads();
  const int n = src < 0 ? 0 : (s_len[src] < keep ? s_len[src] : keep);
  s_n[tid] = n;
  __syncthreads();

  // f(row, page of the row) over rows of ppr pages, four at a time
  auto each = [&](int rows, auto&& load, auto&& use) {
    constexpr int K = 4;
    const int all = rows * ppr, step_row = kSmallThreads / ppr, step_j = kSmallThreads - step_row * ppr;
    int row = tid / ppr, j = tid - row * ppr;
    for (int e = tid; e < all; e += K * kSmallThreads) {
      int rows_of[K], js[K], ids[K];
#pragma unroll
      for (int k = 0; k < K; ++k) {
        rows_of[k] = row;
        js[k] = j;
        ids[k] = e + k * kSmallThreads < all ? load(row, j) : 0;
        row += step_row;
        j += step_j;
        if (j >= ppr) {
          j -= ppr;
          ++row;
        }
      }
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (e + k * kSmallThreads < all) use(rows_of[k], js[k], ids[k], e + k * kSmallThreads);
    }
  };
  each(p.B, [&](int row, int j) { return j < pages_of(s_len[row]) ? p.table[row * ppr + j] : 0; },
       [&](int row, int j, int id, int) {
         if (j >= pages_of(s_len[row])) return;
         if (id < 1 || id > p.cap) ok = false;
         else atomicOr(&word[id], kHeld);
       });
  auto of_source = [&](int row, int j) { return j < pages_of(s_n[row]) ? p.table[s_src[row] * ppr + j] : 0; };
  each(p.R, of_source, [&](int row, int j, int id, int) {
    if (j >= pages_of(s_n[row])) return;
    if (id < 1 || id > p.cap) {
      ok = false;
      return;
    }
    const bool end = (j + 1) * kPage > s_n[row];
    atomicAdd(&word[id], end ? kEnds + 1 : 1u);
    if (end) atomicMax(&begun[id], static_cast<uint32_t>(p.R - row));
  });
  if (!ok) atomicOr(&s_bad, 1u);
  __syncthreads();
  const bool bad = s_bad != 0;

  int last = 0;  // the page that the row goes on writing, where it is not its own
  if (!bad && n % kPage != 0) {
    last = p.table[src * ppr + n / kPage];
    const uint32_t w = word[last];
    if ((w & kCount) == ((w & ~kHeld) / kEnds) && static_cast<int>(begun[last]) == p.R - tid) last = 0;
  }
  int copies, left;
  const int rank = block_scan<kSmallThreads>(last != 0, s_wave, copies);
  s_copy[tid] = last != 0 ? rank : -1;
  const int each_pages = p.cap / kSmallThreads + 1;
  const int id0 = tid * each_pages, id1 = id0 + each_pages <= p.cap + 1 ? id0 + each_pages : p.cap + 1;
  int mine = 0;
  for (int id = id0; id < id1; ++id) mine += is_left(word[id]);
  int to = block_scan<kSmallThreads>(mine, s_wave, left);
  int fail = (bad ? FADE_SLOTS_BAD_COUNT : 0) | before;
  if (head < 0 || head >= p.cap || count < 0 || count > p.cap - left) fail |= FADE_SLOTS_BAD_COUNT;
  else if (copies > count) fail |= FADE_SLOTS_EXHAUSTED;
  if (tid == 0) p.status[0] = fail;
  if (fail) {  // nothing changes
    for (int e = tid; e < p.R * ppr; e += kSmallThreads) p.table_out[e] = e < p.B * ppr ? p.table[e] : 0;
    if (tid < p.R) {
      p.lens_out[tid] = tid < p.B ? p.lens[tid] : 0;
      p.copies[3 * tid] = p.copies[3 * tid + 1] = p.copies[3 * tid + 2] = 0;
    }
    if (tid < 2) p.ring_out[tid] = p.ring[tid];
    return;
  }
  const uint32_t cap = static_cast<uint32_t>(p.cap);
  auto place = [&](int i) { return (static_cast<uint32_t>(head) + static_cast<uint32_t>(i)) % cap; };
  each(p.R, of_source, [&](int row, int j, int id, int e) {
    const int c = s_copy[row];
    p.table_out[e] = c >= 0 && j == s_n[row] / kPage ? p.free_pages[place(c)] : id;
  });
  if (tid < p.R) {
    p.lens_out[tid] = n;
    p.copies[3 * tid] = last;
    p.copies[3 * tid + 1] = last != 0 ? p.free_pages[place(rank)] : 0;
    p.copies[3 * tid + 2] = last != 0 ? n % kPage : 0;
  }
  if (tid == 0) {
    p.ring_out[0] = static_cast<int32_t>(place(copies));
    p.ring_out[1] = count - copies + left;
  }
  if (mine != 0)
    for (int id = id0; id < id1; ++id)
      if (is_left(word[id])) p.free_pages[place(count + to++)] = id;
}

bool is_small(const fade_page_fork_args* a) {
  return a->B <= kSmallRows && a->R <= kSmallRows && a->n_free <= kSmallPages && (a->B + a->R) * a->pages_per_row <= kSmallEntries;
}

int64_t words_of(int64_t cap) { return 2 * (cap + 1) + cap / kSegment + 1 + 2; }

int check_args(const fade_page_fork_args* a, const int32_t* before) {
  const char* what = "fade_page_fork";
  if (a == nullptr) return einval("%s: null args", what);
  if (a->B < 1 || a->B > FADE_SLOTS_MAX_ROWS || a->R < 1 || a->R > FADE_SLOTS_MAX_ROWS)
    return einval("%s: 1 to %d rows, got %lld and %lld", what, FADE_SLOTS_MAX_ROWS, (long long)a->B, (long long)a->R);
  if (a->pages_per_row < 1 || a->pages_per_row > (1 << 24) || (a->B > a->R ? a->B : a->R) * a->pages_per_row >= (1ll << 31))
    return einval("%s: pages_per_row must be 1 to 2^24 with fewer than 2^31 table entries", what);
  if (a->n_free < 1 || a->n_free >= (1ll << 31) / kPage - 1) return einval("%s: bad size of the free ring", what);
  if (!a->lens || !a->table || !a->free_pages || !a->ring || !a->table_out || !a->lens_out || !a->copies || !a->ring_out || !a->status)
    return einval("%s: null pointer", what);
  if (!a->source && a->R != a->B) return einval("%s: without source the rows stay as many as they are", what);
  // what one workgroup writes, others read
  struct Span {
    const void* at;
    int64_t bytes;
    const char* name;
  };
  const Span spans[] = {{a->table_out, 4 * a->R * a->pages_per_row, "table_out"}, {a->lens_out, 4 * a->R, "lens_out"}, {a->copies, 12 * a->R, "copies"},
                        {a->ring_out, 8, "ring_out"}, {a->status, 4, "status"}, {a->free_pages, 4 * a->n_free, "free_pages"},  // (written so far)
                        {a->lens, 4 * a->B, "lens"}, {a->source, a->source ? 4 * a->R : 0, "source"}, {a->keep, a->keep ? 4 * a->R : 0, "keep"},
                        {a->ring, 8, "ring"}, {a->table, 4 * a->B * a->pages_per_row, "table"}, {before, before ? 4 : 0, "before"}};
  for (int i = 0; i < 6; ++i)
    for (int j = i + 1; j < 12; ++j) {
      const uintptr_t x = reinterpret_cast<uintptr_t>(spans[i].at), y = reinterpret_cast<uintptr_t>(spans[j].at);
      if (spans[i].bytes == 0 || spans[j].bytes == 0) continue;
      if (x < y + spans[j].bytes && y < x + spans[i].bytes)
        return einval("%s: %s and %s overlap; what is written must be other memory than the rest of the call's", what, spans[i].name, spans[j].name);
    }
  return FADE_OK;
}

}  // namespace
}  // namespace fork
}  // namespace fade

using namespace fade;

FADE_API int fade_page_fork_workspace_bytes(const fade_page_fork_args* a, int64_t* bytes) {
  if (bytes == nullptr) return einval("fade_page_fork_workspace_bytes: null output");
  const int rc = fade::fork::check_args(a, nullptr);
  if (rc) return rc;
  *bytes = fade::fork::is_small(a) ? 0 : 4 * fade::fork::words_of(a->n_free);
  return FADE_OK;
}

FADE_API int fade_page_fork(const fade_page_fork_args* a, void* workspace, int64_t workspace_bytes, void* stream) {
  return fade_page_fork_after(a, nullptr, workspace, workspace_bytes, stream);
}

FADE_API int fade_page_fork_after(const fade_page_fork_args* a, const int32_t* before, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace fade::fork;
  int rc = check_args(a, before);
  if (rc) return rc;
  const bool small = is_small(a);
  const int64_t words = small ? 0 : words_of(a->n_free);
  if (!small && (workspace == nullptr || workspace_bytes < 4 * words || (reinterpret_cast<uintptr_t>(workspace) & 15)))
    return einval("fade_page_fork: needs a 16-byte aligned workspace of %lld bytes", (long long)(4 * words));
  Params p{};
  p.B = static_cast<int>(a->B);
  p.R = static_cast<int>(a->R);
  p.ppr = static_cast<int>(a->pages_per_row);
  p.cap = static_cast<int>(a->n_free);
  p.lens = a->lens;
  p.source = a->source;
  p.keep = a->keep;
  p.table = a->table;
  p.free_pages = a->free_pages;
  p.ring = a->ring;
  p.before = before;
  p.table_out = a->table_out;
  p.lens_out = a->lens_out;
  p.copies = a->copies;
  p.ring_out = a->ring_out;
  p.status = a->status;
  hipStream_t st = as_stream(stream);
  if (small) {
    hipLaunchKernelGGL(fork_small_kernel, dim3(1), dim3(kSmallThreads), 0, st, p);
    return check_launch("fade_page_fork");
  }
  p.word = static_cast<uint32_t*>(workspace);
  p.first = p.word + p.cap + 1;
  p.left = p.first + p.cap + 1;
  p.bad = p.left + p.cap / kSegment + 1;
  const int64_t most = 2 * static_cast<int64_t>(num_cus());
  auto blocks = [&](int64_t n) { return dim3(static_cast<unsigned>(n < 1 ? 1 : (n > most ? most : n))); };
  const int64_t spans = cdiv(p.ppr, kThreads);
  hipLaunchKernelGGL(fork_clear_kernel, blocks(cdiv(words, 4 * kThreads)), dim3(kThreads), 0, st, p.word, words);
  rc = check_launch("fade_page_fork");
  if (rc) return rc;
  hipLaunchKernelGGL(fork_count_kernel, blocks((a->B + a->R) * spans), dim3(kThreads), 0, st, p);
  rc = check_launch("fade_page_fork");
  if (rc) return rc;
  hipLaunchKernelGGL(fork_left_kernel, dim3(static_cast<unsigned>(p.cap / kSegment + 1)), dim3(kThreads), 0, st, p);
  rc = check_launch("fade_page_fork");
  if (rc) return rc;
  const int64_t items = a->R * spans > p.cap / kSegment + 1 ? a->R * spans : p.cap / kSegment + 1;
  if (a->R <= 256) hipLaunchKernelGGL(fork_write_kernel<256>, blocks(items), dim3(kThreads), 0, st, p);
  else if (a->R <= 1024) hipLaunchKernelGGL(fork_write_kernel<1024>, blocks(items), dim3(kThreads), 0, st, p);
  else hipLaunchKernelGGL(fork_write_kernel<FADE_SLOTS_MAX_ROWS>, blocks(items), dim3(kThreads), 0, st, p);
  return check_launch("fade_page_fork");
}
