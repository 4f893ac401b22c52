// Trees of drafted tokens: what each token sees, its depth and its position.
//
// A row's tokens are numbered so that every token follows an earlier one (or none).
// Token i sees itself and what the token that it follows sees; its depth is the number
// of tokens on the way up.  A thread takes one word of one token's mask and goes up the
// parents, which lie in LDS: a way ends early where only tokens below the word's are left.
// Bound by latency: the row's counts, its parents, the steps up, the writes (12 tokens of
// one row 2.4 us, 256 rows of 64 3.3).
#include "fade_common.h"

namespace fade {
namespace {

constexpr int kThreads = 256;

__global__ __launch_bounds__(kThreads) void draft_tree_kernel(fade_draft_tree_args p) {
  __shared__ int16_t up[FADE_DRAFT_MAX_NODES];
  __shared__ int32_t s_bad;
  const int b = blockIdx.x, T = static_cast<int>(p.T), words = static_cast<int>(p.words);
  int s = p.starts[b], e = p.starts[b + 1];
  s = s < 0 ? 0 : (s > T ? T : s);
  e = e < s ? s : (e > T ? T : e);
  const int n = e - s, known = n < 32 * words ? n : 32 * words;
  const int base = static_cast<int>(static_cast<uint32_t>(p.lens[b]) - static_cast<uint32_t>(n));
  if (threadIdx.x == 0) s_bad = n > known ? FADE_DRAFT_TOO_MANY : 0;
  __syncthreads();
  for (int i = threadIdx.x; i < known; i += kThreads) {
    int u = p.parents[s + i];
    if (u < -1 || u >= i) {
      atomicOr(&s_bad, FADE_DRAFT_BAD_PARENT);
      u = -1;
    }
    up[i] = static_cast<int16_t>(u);
  }
  __syncthreads();
  if (threadIdx.x == 0) p.status[b] = s_bad;
  for (int64_t x = threadIdx.x; x < static_cast<int64_t>(n) * words; x += kThreads) {
    const int i = static_cast<int>(x / words), w = static_cast<int>(x - static_cast<int64_t>(i) * words);
    uint32_t bits = 0;
    int depth = -1;  // (of word 0, whose thread goes all the way up)
    if (i < known)
      for (int j = i; j >= 32 * w; j = up[j]) {
        if (j >> 5 == w) bits |= 1u << (j & 31);
        ++depth;
      }
    p.bits[(static_cast<int64_t>(s) + i) * words + w] = bits;
    if (w == 0) {
      depth = depth < 0 ? 0 : depth;
      p.depth[s + i] = depth;
      p.positions[s + i] = base + depth;
    }
  }
  int end = p.starts[p.B];
  end = end < 0 ? 0 : end;
  for (int64_t t = static_cast<int64_t>(end) + b; t < T; t += p.B) {
    for (int w = threadIdx.x; w < words; w += kThreads) p.bits[t * words + w] = 0;
    if (threadIdx.x == 0) p.depth[t] = p.positions[t] = 0;
  }
}

}  // namespace
}  // namespace fade

using namespace fade;

FADE_API int fade_draft_tree(const fade_draft_tree_args* a, void* stream) {
  if (a == nullptr) return einval("fade_draft_tree: null args");
  if (a->B < 1 || a->B > (1 << 20) || a->T < 0 || a->T > (1 << 24)) return einval("fade_draft_tree: B must be 1 to 2^20, T 0 to 2^24");
  if (a->words < 1 || a->words > FADE_DRAFT_MAX_NODES / 32)
    return einval("fade_draft_tree: words must be 1 to %d, got %lld", FADE_DRAFT_MAX_NODES / 32, (long long)a->words);
  if (!a->lens || !a->starts || !a->status || (a->T > 0 && (!a->parents || !a->bits || !a->depth || !a->positions)))
    return einval("fade_draft_tree: null pointer");
  hipLaunchKernelGGL(draft_tree_kernel, dim3(static_cast<unsigned>(a->B)), dim3(kThreads), 0, as_stream(stream), *a);
  return check_launch("fade_draft_tree");
}
