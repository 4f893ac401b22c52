// Block tables and slot maps of a paged cache, built on the GPU from the rows'
// token counts.
//
// Row b holds lens[b] tokens and gets new[b] more; a row with reset[b] starts
// anew (its pages go back to the free ones, its tokens count from 0).  With
// pages(x) = ceil(x / 64), held_b = lens[b] (0 for a row that starts anew) and
// need_b = pages(held_b + new_b) - pages(held_b), page j >= pages(held_b) of row b
// is the free page number sum_{a < b} need_a + j - pages(held_b), and token i of the
// row's new ones sits at position held_b + i, slot 64 * page + position % 64.
// Free pages are a ring: taken at its head, put back behind its tail.  What this
// call puts back lies outside what it takes, so nothing waits for another
// workgroup, and a call repeated on the same inputs writes the same values.
//
// One launch.  Every workgroup sums the counts of all rows by itself (in LDS: the
// rows' token starts, page starts and returned-page starts) and then writes its
// share of the outputs: entries of the table and slots of the new tokens.  What
// bounds it is latency (the counts' loads, the sums' barriers, a token's search
// and table read), not the bytes: 16 rows of 512 pages 4.0 us, 1000 rows of 1024
// pages with 16 chunks 7.9 (8 MB, 1.2 us at a large copy's rate), 4096 rows of 256
// pages 20.8, of 16 pages 20.4.
#include "fade_common.h"

namespace fade {
namespace {

constexpr int kPage = 64;
constexpr int kThreads = 256;

struct SlotParams {
  int B, ppr, n_tokens, cap;
  int wide;  // table rows are whole aligned groups of four entries
  const int32_t* lens;
  const int32_t* fresh;
  const uint8_t* reset;
  const int32_t* table;
  int32_t* free_pages;
  const int32_t* ring;
  int32_t* table_out;
  int32_t* lens_out;
  int32_t* starts;
  int32_t* slots;
  int32_t* positions;
  int32_t* ring_out;
  int32_t* status;
};

__device__ __forceinline__ int pages_of(int tokens) { return (tokens + (kPage - 1)) / kPage; }

// ROWS: the most rows of the instance.
template <int ROWS>
__global__ __launch_bounds__(kThreads) void page_slots_kernel(SlotParams p) {
  constexpr int PER = ROWS / kThreads;  // rows per thread
  __shared__ int32_t s_start[ROWS + 1];  // first new token of a row
  __shared__ int32_t s_need[ROWS + 1];   // its first free page, counted from the head
  __shared__ int32_t s_back[ROWS + 1];   // the first place behind the tail for its returned pages
  __shared__ int32_t s_lens[ROWS];       // tokens held; ~tokens where the row starts anew
  __shared__ int64_t s_wave[2][kThreads / 64];
  __shared__ int32_t s_bad;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row_cap = static_cast<int64_t>(p.ppr) * kPage;
  if (tid == 0) s_bad = 0;
  __syncthreads();

  // this thread's rows tid * PER ..: their counts, summed over the workgroup (tokens
  // in 64 bits; needed and returned pages, at most B * ppr < 2^31 each, side by side)
  int n_tok[PER], n_need[PER], n_back[PER];
  int64_t tok = 0, pg = 0;
  int bad = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int b = tid * PER + i;
    n_tok[i] = n_need[i] = n_back[i] = 0;
    if (b < p.B) {
      int held = p.lens[b], add = p.fresh[b];
      const bool again = p.reset != nullptr && p.reset[b] != 0;
      if (held < 0 || held > row_cap || add < 0) {
        bad |= FADE_SLOTS_BAD_COUNT;
        held = add = 0;
      }
      const int from = again ? 0 : held;
      if (from + static_cast<int64_t>(add) > row_cap) {
        bad |= FADE_SLOTS_ROW_FULL;
        add = 0;
      }
      s_lens[b] = again ? ~held : held;
      n_tok[i] = add;
      n_need[i] = pages_of(from + add) - pages_of(from);
      n_back[i] = again ? pages_of(held) : 0;
      tok += n_tok[i];
      pg += (static_cast<int64_t>(n_back[i]) << 32) + n_need[i];
    }
  }
  if (bad) atomicOr(&s_bad, bad);
  int64_t it = tok, ip = pg;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t a = __shfl_up(it, o, 64), c = __shfl_up(ip, o, 64);
    if (lane >= o) {
      it += a;
      ip += c;
    }
  }
  if (lane == 63) {
    s_wave[0][wave] = it;
    s_wave[1][wave] = ip;
  }
  __syncthreads();
  int64_t all_tok = 0, all_pg = 0;
  it -= tok;
  ip -= pg;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    if (w < wave) {
      it += s_wave[0][w];
      ip += s_wave[1][w];
    }
    all_tok += s_wave[0][w];
    all_pg += s_wave[1][w];
  }
  const int need = static_cast<int>(all_pg & 0xFFFFFFFF), back = static_cast<int>(all_pg >> 32);
  const int head = p.ring[0], count = p.ring[1];
  int fail = s_bad;
  if (head < 0 || head >= p.cap || count < 0 || count > p.cap - back) fail |= FADE_SLOTS_BAD_COUNT;
  else if (need > count) fail |= FADE_SLOTS_EXHAUSTED;
  if (all_tok > p.n_tokens) fail |= FADE_SLOTS_TOO_MANY;
  int64_t rt = it, rp = ip;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int b = tid * PER + i;
    if (b < p.B) {
      s_start[b] = static_cast<int32_t>(rt);
      s_need[b] = static_cast<int32_t>(rp & 0xFFFFFFFF);
      s_back[b] = static_cast<int32_t>(rp >> 32);
    }
    rt += n_tok[i];
    rp += (static_cast<int64_t>(n_back[i]) << 32) + n_need[i];
  }
  if (tid == 0) {
    s_start[p.B] = static_cast<int32_t>(all_tok);
    s_need[p.B] = need;
    s_back[p.B] = back;
  }
  __syncthreads();

  const int64_t stride = static_cast<int64_t>(gridDim.x) * kThreads;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kThreads + tid;
  if (fail) {  // nothing changes
    for (int64_t e = first; e < static_cast<int64_t>(p.B) * p.ppr; e += stride) p.table_out[e] = p.table[e];
    for (int64_t t = first; t < p.n_tokens; t += stride) {
      p.slots[t] = -1;
      p.positions[t] = 0;
    }
    for (int64_t b = first; b < p.B; b += stride) p.lens_out[b] = p.lens[b];
    for (int64_t b = first; b <= p.B; b += stride) p.starts[b] = 0;
    if (first == 0) {
      p.ring_out[0] = head;
      p.ring_out[1] = count;
      p.status[0] = fail;
    }
    return;
  }
  // free page number j from the head, place j behind the tail (sums below 2^32)
  const uint32_t cap = static_cast<uint32_t>(p.cap);
  auto taken = [&](int j) { return p.free_pages[(static_cast<uint32_t>(head) + static_cast<uint32_t>(j)) % cap]; };
  // The table: a workgroup takes a row's next 1024 (256) entries, four (one) a thread (1000 rows of 1024 entries 7.5 us,
  // one a thread 8.9).
  auto entry = [&](int j, int old, int have, int mine, int need0, int back0, bool again, int was) {
    if (again && j < old) p.free_pages[(static_cast<uint64_t>(head) + count + back0 + j) % cap] = was;
    return j >= have && j < have + mine ? taken(need0 + j - have) : (j < have ? was : 0);
  };
  const int span = p.wide ? 4 * kThreads : kThreads;
  const int spans = (p.ppr + span - 1) / span;
  for (int64_t item = blockIdx.x; item < static_cast<int64_t>(p.B) * spans; item += gridDim.x) {
    const int b = spans == 1 ? static_cast<int>(item) : static_cast<int>(item / spans);
    const int j0 = (static_cast<int>(item) - b * spans) * span;
    const int raw = s_lens[b], old = pages_of(raw < 0 ? ~raw : raw), have = raw < 0 ? 0 : old;
    const int need0 = s_need[b], mine = s_need[b + 1] - need0, back0 = s_back[b];
    const int64_t at = static_cast<int64_t>(b) * p.ppr;
    if (p.wide) {
      const int j = j0 + 4 * tid;
      if (j >= p.ppr) continue;
      int4 was = make_int4(0, 0, 0, 0);
      if (j < old) was = *reinterpret_cast<const int4*>(p.table + at + j);
      int4 id = make_int4(0, 0, 0, 0);
      if (j < old || j < have + mine) {
        id.x = entry(j, old, have, mine, need0, back0, raw < 0, was.x);
        id.y = entry(j + 1, old, have, mine, need0, back0, raw < 0, was.y);
        id.z = entry(j + 2, old, have, mine, need0, back0, raw < 0, was.z);
        id.w = entry(j + 3, old, have, mine, need0, back0, raw < 0, was.w);
      }
      *reinterpret_cast<int4*>(p.table_out + at + j) = id;
    } else {
      const int j = j0 + tid;
      if (j >= p.ppr) continue;
      p.table_out[at + j] = entry(j, old, have, mine, need0, back0, raw < 0, j < old ? p.table[at + j] : 0);
    }
  }
  for (int64_t t = first; t < p.n_tokens; t += stride) {
    int slot = -1, pos = 0;
    if (t < all_tok) {
      // the last row that starts at or before t
      int lo = 0, hi = p.B;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_start[mid] <= t) lo = mid;
        else hi = mid;
      }
      const int raw = s_lens[lo], from = raw < 0 ? 0 : raw, have = pages_of(from);
      pos = from + static_cast<int>(t) - s_start[lo];
      const int j = pos / kPage;
      const int id = j < have ? p.table[static_cast<int64_t>(lo) * p.ppr + j] : taken(s_need[lo] + j - have);
      slot = id * kPage + pos % kPage;
    }
    p.slots[t] = slot;
    p.positions[t] = pos;
  }
  for (int64_t b = first; b <= p.B; b += stride) {
    p.starts[b] = s_start[b];
    if (b < p.B) p.lens_out[b] = (s_lens[b] < 0 ? 0 : s_lens[b]) + s_start[b + 1] - s_start[b];
  }
  if (first == 0) {
    p.ring_out[0] = static_cast<int32_t>((static_cast<uint32_t>(head) + static_cast<uint32_t>(need)) % cap);
    p.ring_out[1] = count - need + back;
    p.status[0] = 0;
  }
}

}  // namespace
}  // namespace fade

using namespace fade;

FADE_API int fade_page_slots(const fade_page_slots_args* a, void* stream) {
  if (a == nullptr) return einval("fade_page_slots: null args");
  if (a->B < 1 || a->B > FADE_SLOTS_MAX_ROWS)
    return einval("fade_page_slots: 1 to %d rows, got %lld", FADE_SLOTS_MAX_ROWS, (long long)a->B);
  if (a->pages_per_row < 1 || a->pages_per_row > (1 << 24) || a->B * a->pages_per_row >= (1ll << 31))
    return einval("fade_page_slots: pages_per_row must be 1 to 2^24 with fewer than 2^31 table entries");
  if (a->n_tokens < 0 || a->n_tokens >= (1ll << 31)) return einval("fade_page_slots: n_tokens must be 0 to 2^31 - 1");
  if (a->n_free < 1 || a->n_free >= (1ll << 31) / kPage - 1) return einval("fade_page_slots: bad size of the free ring");
  if (!a->lens || !a->new_tokens || !a->table || !a->free_pages || !a->ring || !a->table_out || !a->lens_out || !a->starts ||
      !a->ring_out || !a->status || (a->n_tokens > 0 && (!a->slots || !a->positions)))
    return einval("fade_page_slots: null pointer");
  // what one workgroup writes, others read: every array of the call has memory of its own, but table_out may be table
  // (a workgroup reads the entries that it writes, and those of a row's pages, which stay as they are)
  struct Span {
    const void* at;
    int64_t bytes;
    const char* name;
  };
  const Span spans[] = {{a->table_out, 4 * a->B * a->pages_per_row, "table_out"}, {a->lens_out, 4 * a->B, "lens_out"},
                        {a->starts, 4 * a->B + 4, "starts"}, {a->slots, 4 * a->n_tokens, "slots"},
                        {a->positions, 4 * a->n_tokens, "positions"}, {a->ring_out, 8, "ring_out"}, {a->status, 4, "status"},
                        {a->free_pages, 4 * a->n_free, "free_pages"},  // (written so far)
                        {a->lens, 4 * a->B, "lens"}, {a->new_tokens, 4 * a->B, "new_tokens"}, {a->reset, a->reset ? a->B : 0, "reset"},
                        {a->ring, 8, "ring"}, {a->table, 4 * a->B * a->pages_per_row, "table"}};
  for (int i = 0; i < 8; ++i)
    for (int j = i + 1; j < 13; ++j) {
      const uintptr_t x = reinterpret_cast<uintptr_t>(spans[i].at), y = reinterpret_cast<uintptr_t>(spans[j].at);
      if ((i == 0 && j == 12 && x == y) || spans[i].bytes == 0 || spans[j].bytes == 0) continue;
      if (x < y + spans[j].bytes && y < x + spans[i].bytes)
        return einval("fade_page_slots: %s and %s overlap; what is written must be other memory than the rest of the call's (table_out may be table)",
                      spans[i].name, spans[j].name);
    }
  SlotParams p;
  p.B = static_cast<int>(a->B);
  p.ppr = static_cast<int>(a->pages_per_row);
  p.n_tokens = static_cast<int>(a->n_tokens);
  p.cap = static_cast<int>(a->n_free);
  p.lens = a->lens;
  p.fresh = a->new_tokens;
  p.reset = a->reset;
  p.table = a->table;
  p.free_pages = a->free_pages;
  p.ring = a->ring;
  p.table_out = a->table_out;
  p.lens_out = a->lens_out;
  p.starts = a->starts;
  p.slots = a->slots;
  p.positions = a->positions;
  p.ring_out = a->ring_out;
  p.status = a->status;
  p.wide = p.ppr % 4 == 0 && ((reinterpret_cast<uintptr_t>(a->table) | reinterpret_cast<uintptr_t>(a->table_out)) & 15) == 0;
  const int64_t items = a->B * cdiv(p.ppr, p.wide ? 4 * kThreads : kThreads);
  int64_t blocks = items > cdiv(a->n_tokens, kThreads) ? items : cdiv(a->n_tokens, kThreads);
  if (blocks > 2 * num_cus()) blocks = 2 * num_cus();
  const dim3 grid(static_cast<unsigned>(blocks));
  // The fewer rows an instance has, the less LDS it takes and the shorter its sums are (in the one of 4096 rows
  // 16 rows take 7.5 us instead of 4.0, 1000 rows 11.3 instead of 7.5).
  if (a->B <= 256) hipLaunchKernelGGL(page_slots_kernel<256>, grid, dim3(kThreads), 0, as_stream(stream), p);
  else if (a->B <= 1024) hipLaunchKernelGGL(page_slots_kernel<1024>, grid, dim3(kThreads), 0, as_stream(stream), p);
  else hipLaunchKernelGGL(page_slots_kernel<FADE_SLOTS_MAX_ROWS>, grid, dim3(kThreads), 0, as_stream(stream), p);
  return check_launch("fade_page_slots");
}
