// Drafted tokens against the target's probabilities, without a change of the target's
// distribution.
//
// The walk starts at a row's token 0.  A child x of the token where it stands is accepted
// where a uniform number says so, else refused, and the next child is tried on what is left:
//   children drawn from q: a_0 = p, a_{k+1} = max(a_k - q, 0) / its sum.  By induction
//     a_k = max(p - s_k q, 0) / N_k  with  s_0 = 0, N_0 = 1, s_{k+1} = s_k + N_k,
//     N_k = sum max(p - s_k q, 0):
//   one number describes what is left, and a refusal costs one pass over the vocabulary (none
//   the last one at a token: the next token's drawing sums as well).  x is accepted where
//   u N_k q_x < max(p_x - s_k q_x, 0).
//   children chosen without chance: what is left is p without the refused tokens, its sum
//     1 less their probabilities.
// Where no child is accepted, the next token is the first at which the running sum of what is
// left passes its share of the sum: sums over segments of the vocabulary, then over parts of
// the segment that holds the place, then token by token.  All sums are in 64 bits: with 1e5
// tokens, 32 would move one drawing in a hundred to a neighbour.
#include "fade_common.h"

namespace fade {
namespace verify {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kMaxNodes = FADE_DRAFT_MAX_NODES;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <typename E>
__device__ __forceinline__ float prob(E x) {
  const float f = to_f32(x);
  return f > 0.0f ? f : 0.0f;  // (a NaN too)
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// What the tests of a row's tokens need, in LDS.
struct Nodes {
  int16_t up[kMaxNodes];
  int32_t tok[kMaxNodes];  // -1: outside the vocabulary
  float p[kMaxNodes], q[kMaxNodes], u[kMaxNodes];
};

// What is left of a token's probabilities.
template <typename E>
struct Rest {
  const E* p;
  const E* q;    // or null
  int V;
  double s;      // q's share
  const Nodes* nodes;
  int n, refused_of;  // refused: the children of that token (-1: none)
};

constexpr int kBatch = 4;  // tiles whose loads are in flight together

// A lane's VEC elements from i on of a row, as bits; zeros past `end`.
template <typename E>
__device__ __forceinline__ u32x4 load_bits(const E* row, int i, int end) {
  constexpr int VEC = 16 / sizeof(E);
  u32x4 r = {0, 0, 0, 0};
  if (i + VEC <= end) {
    __builtin_memcpy(&r, row + i, 16);
  } else if (i < end) {
    E e[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) e[j] = E{};
#pragma unroll
    for (int j = 0; j < VEC; ++j)
      if (i + j < end) e[j] = row[i + j];
    __builtin_memcpy(&r, e, 16);
  }
  return r;
}

// The weights of a lane's VEC tokens from i on; the wave's tile starts at `tile`.
// All lanes call it.
template <typename E>
__device__ __forceinline__ void weights(const Rest<E>& r, u32x4 pb, u32x4 qb, int i, int tile, double (&w)[16 / sizeof(E)]) {
  constexpr int VEC = 16 / sizeof(E);
  E pe[VEC], qe[VEC];
  __builtin_memcpy(pe, &pb, 16);
  __builtin_memcpy(qe, &qb, 16);
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    const double x = prob(pe[j]);
    const double y = r.s > 0.0 ? fma(-r.s, static_cast<double>(prob(qe[j])), x) : x;
    w[j] = y > 0.0 ? y : 0.0;
  }
  if (r.refused_of < 0) return;
  const int lane = threadIdx.x & 63;
  for (int c0 = r.refused_of + 1; c0 < r.n; c0 += 64) {
    const int c = c0 + lane;
    const int x = c < r.n && r.nodes->up[c] == r.refused_of ? r.nodes->tok[c] : -1;
    uint64_t hit = __builtin_amdgcn_ballot_w64(x >= tile && x < tile + 64 * VEC);
    while (hit != 0) {
      const int at = __builtin_amdgcn_readlane(x, __builtin_ctzll(hit)) - i;
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (at == j) w[j] = 0.0;
      hit &= hit - 1;
    }
  }
}

// A wave's sum of the weights of tokens i0 .. i1 - 1.
template <typename E>
__device__ double range_sum(const Rest<E>& r, int i0, int i1) {
  constexpr int VEC = 16 / sizeof(E), TILE = 64 * VEC;
  const int lane = threadIdx.x & 63;
  const bool two = r.s > 0.0;
  double acc = 0.0;
  for (int t0 = i0; t0 < i1; t0 += kBatch * TILE) {
    u32x4 pb[kBatch], qb[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int i = t0 + k * TILE + VEC * lane;
      pb[k] = load_bits(r.p, i, i1);
      qb[k] = two ? load_bits(r.q, i, i1) : u32x4{0, 0, 0, 0};
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      if (t0 + k * TILE >= i1) break;
      double w[VEC];
      weights(r, pb[k], qb[k], t0 + k * TILE + VEC * lane, t0 + k * TILE, w);
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc += w[j];
    }
  }
  return wave_sum(acc);
}

// The first token of i0 .. i1 - 1 at which `before` plus the running sum passes t, else the
// last with a weight, else -1.  One wave.
template <typename E>
__device__ int find_token(const Rest<E>& r, int i0, int i1, double before, double t) {
  constexpr int VEC = 16 / sizeof(E), TILE = 64 * VEC;
  const int lane = threadIdx.x & 63;
  int last = -1;
  for (int t0 = i0; t0 < i1; t0 += TILE) {
    const int i = t0 + VEC * lane;
    double w[VEC], own = 0.0;
    weights(r, load_bits(r.p, i, i1), r.s > 0.0 ? load_bits(r.q, i, i1) : u32x4{0, 0, 0, 0}, i, t0, w);
#pragma unroll
    for (int j = 0; j < VEC; ++j) own += w[j];
    double upto = own;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double x = __shfl_up(upto, o, 64);
      if (lane >= o) upto += x;
    }
    const double total = __shfl(upto, 63, 64);
    double c = before + (upto - own);
    int found = -1, any = -1;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      c += w[j];
      if (w[j] > 0.0) {
        any = i + j;
        if (found < 0 && c > t) found = i + j;
      }
    }
    const uint64_t hit = __builtin_amdgcn_ballot_w64(found >= 0), some = __builtin_amdgcn_ballot_w64(any >= 0);
    if (hit != 0) return __builtin_amdgcn_readlane(found, __builtin_ctzll(hit));
    if (some != 0) last = __builtin_amdgcn_readlane(any, 63 - __builtin_clzll(some));
    before += total;
  }
  return last;
}

// A row's walk; the same in every wave that makes it.
struct Walk {
  int cur, last, count, tried;  // token, the last child tried, tokens of the path, children refused at cur
  double s, norm;
  bool sum;   // stands before a child that needs the sum of what is left
  bool done;
};

template <typename E>
__global__ __launch_bounds__(kThreads) void verify_kernel(fade_verify_args a) {
  __shared__ Nodes nodes;
  __shared__ double sums[kWaves];
  __shared__ int answer;
  const int b = blockIdx.x, T = static_cast<int>(a.T), V = static_cast<int>(a.V);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int s = a.starts[b], e = a.starts[b + 1];
  s = s < 0 ? 0 : (s > T ? T : s);
  e = e < s ? s : (e > T ? T : e);
  const int n = e - s < kMaxNodes ? e - s : kMaxNodes;
  const E* const target = static_cast<const E*>(a.target);
  const E* const draft = static_cast<const E*>(a.draft);
  const int64_t out0 = static_cast<int64_t>(b) * a.max_path;
  auto put_token = [&](void* to, int64_t at, int64_t x) {
    if (a.tok64) static_cast<int64_t*>(to)[at] = x;
    else static_cast<int32_t*>(to)[at] = static_cast<int32_t>(x);
  };
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int up = i == 0 ? -1 : a.parents[s + i];
    const int64_t x = a.tok64 ? static_cast<const int64_t*>(a.tokens)[s + i] : static_cast<const int32_t*>(a.tokens)[s + i];
    const bool ok = up >= 0 && up < i && x >= 0 && x < V;
    nodes.up[i] = static_cast<int16_t>(up >= 0 && up < i ? up : -1);
    nodes.tok[i] = x >= 0 && x < V ? static_cast<int32_t>(x) : -1;
    nodes.u[i] = a.uniforms[s + i];
    nodes.p[i] = ok ? prob(target[(static_cast<int64_t>(s) + up) * a.target_st + x]) : 0.0f;
    nodes.q[i] = ok && draft != nullptr ? prob(draft[(static_cast<int64_t>(s) + up) * a.draft_st + x]) : 0.0f;
  }
  __syncthreads();
  auto rest = [&](int cur, double share, int refused_of) {
    Rest<E> r;
    r.p = target + (static_cast<int64_t>(s) + cur) * a.target_st;
    r.q = draft == nullptr ? nullptr : draft + (static_cast<int64_t>(s) + cur) * a.draft_st;
    r.V = V;
    r.s = share;
    r.nodes = &nodes;
    r.n = n;
    r.refused_of = refused_of;
    return r;
  };
  // sums of the segments, one a wave
  constexpr int TILE = 64 * (16 / sizeof(E));
  const int seg = (V + kWaves * TILE - 1) / (kWaves * TILE) * TILE;
  auto total = [&](const Rest<E>& r) {
    const int i0 = wave * seg, i1 = i0 + seg < V ? i0 + seg : V;
    const double x = i0 < V ? range_sum(r, i0, i1) : 0.0;
    __syncthreads();
    if (lane == 0) sums[wave] = x;
    __syncthreads();
    double all = 0.0;
    for (int i = 0; i < kWaves; ++i) all += sums[i];
    return all;
  };

  Walk k{0, 0, n > 0 ? 1 : 0, 0, 0.0, 1.0, false, n == 0};
  if (n > 0 && threadIdx.x == 0) a.path[out0] = 0;
  while (!k.done) {
    // the next child of cur
    int c = -1;
    if (k.count < a.max_path)
      for (int c0 = k.last + 1; c0 < n; c0 += 64) {
        const uint64_t who = __builtin_amdgcn_ballot_w64(c0 + lane < n && nodes.up[c0 + lane] == k.cur);
        if (who != 0) {
          c = c0 + __builtin_ctzll(who);
          break;
        }
      }
    if (c < 0) break;
    if (draft != nullptr && k.tried > 0) k.norm = total(rest(k.cur, k.s, -1));
    double left, bound;
    if (draft != nullptr) {
      left = fma(-k.s, static_cast<double>(nodes.q[c]), static_cast<double>(nodes.p[c]));
      bound = static_cast<double>(nodes.u[c]) * k.norm * nodes.q[c];
    } else {
      bool again = false;  // refused already
      for (int c0 = k.cur + 1; c0 < c; c0 += 64)
        again |= __builtin_amdgcn_ballot_w64(c0 + lane < c && nodes.up[c0 + lane] == k.cur && nodes.tok[c0 + lane] == nodes.tok[c]) != 0;
      left = again ? 0.0 : nodes.p[c];
      bound = nodes.u[c] * k.norm;
    }
    k.last = c;
    if (left > 0.0 && bound < left) {
      if (threadIdx.x == 0) {
        a.path[out0 + k.count] = c;
        put_token(a.tokens_out, out0 + k.count - 1, nodes.tok[c]);
      }
      k.cur = c;
      ++k.count;
      k.tried = 0;
      k.s = 0.0;
      k.norm = 1.0;
    } else {
      ++k.tried;
      if (draft != nullptr) k.s += k.norm;
      else k.norm -= left > 0.0 ? left : 0.0;
    }
  }

  int next = -1;
  if (n > 0) {
    Rest<E> r = rest(k.cur, k.s, draft == nullptr && k.tried > 0 ? k.cur : -1);
    double all = total(r);
    if (!(all > 0.0)) {
      r = rest(k.cur, 0.0, -1);
      all = total(r);
    }
    if (all > 0.0) {
      const double t = static_cast<double>(a.final_u[b]) * all;
      // the segment, then the part of it, then the token
      int i0 = 0, i1 = V;
      double before = 0.0;
      auto narrow = [&](int part) {
        int at = -1, full = 0;
        double c = before, c_full = before;
        for (int i = 0; i < kWaves; ++i) {
          if (sums[i] > 0.0) {
            full = i;
            c_full = c;
            if (c + sums[i] > t) {
              at = i;
              break;
            }
          }
          c += sums[i];
        }
        if (at < 0) at = full;  // (the last with a weight)
        before = c_full;
        i0 += at * part;
        i1 = i0 + part < i1 ? i0 + part : i1;
      };
      narrow(seg);
      const int part = ((i1 - i0) + kWaves * TILE - 1) / (kWaves * TILE) * TILE;
      const int j0 = i0 + wave * part, j1 = j0 + part < i1 ? j0 + part : i1;
      const double x = j0 < i1 ? range_sum(r, j0, j1) : 0.0;
      __syncthreads();
      if (lane == 0) sums[wave] = x;
      __syncthreads();
      narrow(part);
      if (wave == 0) answer = find_token(r, i0, i1, before, t);
      __syncthreads();
      next = answer;
    }
  }
  for (int i = k.count + threadIdx.x; i < a.max_path; i += kThreads) a.path[out0 + i] = -1;
  for (int i = (k.count > 0 ? k.count : 0) + threadIdx.x; i < a.max_path; i += kThreads) put_token(a.tokens_out, out0 + i, -1);
  if (threadIdx.x == 0) {
    if (k.count > 0) put_token(a.tokens_out, out0 + k.count - 1, next);
    a.counts[b] = k.count;
    put_token(a.next, b, next);
  }
}

int check_args(const fade_verify_args* a) {
  const char* what = "fade_verify_drafts";
  if (a == nullptr) return einval("%s: null args", what);
  if (a->B < 1 || a->B > (1 << 20) || a->T < 0 || a->T > (1 << 24)) return einval("%s: B must be 1 to 2^20, T 0 to 2^24", what);
  if (a->V < 1 || a->V > (1 << 24)) return einval("%s: V must be 1 to 2^24, got %lld", what, (long long)a->V);
  if (a->max_path < 1 || a->max_path > FADE_DRAFT_MAX_NODES)
    return einval("%s: max_path must be 1 to %d, got %lld", what, FADE_DRAFT_MAX_NODES, (long long)a->max_path);
  if (a->dtype != FADE_DTYPE_F16 && a->dtype != FADE_DTYPE_BF16 && a->dtype != FADE_DTYPE_F32)
    return einval("%s: dtype must be FADE_DTYPE_F16, BF16 or F32, got %d", what, a->dtype);
  if (a->target_st < 0 || (a->draft && a->draft_st < 0)) return einval("%s: negative strides", what);
  if (!a->starts || !a->final_u || !a->path || !a->counts || !a->tokens_out || !a->next ||
      (a->T > 0 && (!a->target || !a->tokens || !a->parents || !a->uniforms)))
    return einval("%s: null pointer", what);
  return FADE_OK;
}

}  // namespace
}  // namespace verify
}  // namespace fade

using namespace fade;
using namespace fade::verify;

FADE_API int fade_verify_workspace_bytes(const fade_verify_args* a, int64_t* bytes) {
  if (bytes == nullptr) return einval("fade_verify_workspace_bytes: null output");
  const int rc = check_args(a);
  if (rc) return rc;
  *bytes = 0;
  return FADE_OK;
}

FADE_API int fade_verify_drafts(const fade_verify_args* a, void* workspace, int64_t workspace_bytes, void* stream) {
  const int rc = check_args(a);
  if (rc) return rc;
  const dim3 grid(static_cast<unsigned>(a->B));
  if (a->dtype == FADE_DTYPE_F32) hipLaunchKernelGGL(verify_kernel<float>, grid, dim3(kThreads), 0, as_stream(stream), *a);
  else if (a->dtype == FADE_DTYPE_BF16) hipLaunchKernelGGL(verify_kernel<Bf16>, grid, dim3(kThreads), 0, as_stream(stream), *a);
  else hipLaunchKernelGGL(verify_kernel<uint16_t>, grid, dim3(kThreads), 0, as_stream(stream), *a);
  return check_launch("fade_verify_drafts");
}
