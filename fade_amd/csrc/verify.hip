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
//
// Bound by latency: a row's counts, its tokens and their probabilities, the walk (64 tokens in
// the lanes' registers), then for each sum a pass over its part of the vocabulary, the exchange
// (about 3 us a sum together), and three narrower passes to the token.  On the GPU: a chain of five tokens
// of one row over 32000 tokens 9.5 us, 48 rows over 128256 without draft probabilities 14 (2.4
// at a copy's rate), 32 trees drawn from a draft over 152064, four or five sums in the longest
// row, 24 (7.6).  128 rows over 152064 tokens 32 (30).
#include "fade_common.h"

namespace fade {
namespace verify {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kMaxNodes = FADE_DRAFT_MAX_NODES;

template <typename E>
__device__ __forceinline__ float prob(E x) {
  return fmaxf(to_f32(x), 0.0f);  // (of a NaN too)
}

// Sums over the wave's lanes up to each one: shifts within rows of 16 lanes, then each row's
// last lane to the next rows (DPP: no LDS round trips).
template <int CTRL, int ROWS>
__device__ __forceinline__ double scan_step(double v) {
  const uint64_t x = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(x), CTRL, ROWS, 0xF, true);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(x >> 32), CTRL, ROWS, 0xF, true);
  return v + __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
__device__ __forceinline__ double wave_scan(double v) {
  v = scan_step<0x111, 0xF>(v);  // row_shr 1, 2, 4, 8
  v = scan_step<0x112, 0xF>(v);
  v = scan_step<0x114, 0xF>(v);
  v = scan_step<0x118, 0xF>(v);
  v = scan_step<0x142, 0xA>(v);  // row_bcast 15 to rows 1 and 3
  return scan_step<0x143, 0xC>(v);  // row_bcast 31 to rows 2 and 3
}
__device__ __forceinline__ double of_lane(double v, int l) {
  const uint64_t x = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(x), l), hi = __builtin_amdgcn_readlane(static_cast<int>(x >> 32), l);
  return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
__device__ __forceinline__ float of_lane(float x, int l) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), l)); }

// What the tests of a row's tokens need, in LDS.
struct Nodes {
  int16_t up[kMaxNodes];
  int32_t tok[kMaxNodes];  // -1: outside the vocabulary (then up is -1 too)
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
  int mine;           // the lane's one of the first 64 after it (-1: none)
};

// A batch of a wave's tiles from t0 on, VEC tokens a lane, as bits.  A lane past the end of the row
// reads the row's last VEC tokens, some of which are others' or its own further on.
constexpr int kBatch = 4;
template <typename E, int VEC>
struct Batch {
  static constexpr int TILE = 64 * VEC;
  struct __attribute__((packed)) Bits {
    E e[VEC];
  };
  Bits p[kBatch], q[kBatch];
  static __device__ __forceinline__ int from(int i, int V) { return i < V - VEC ? i : V - VEC; }
  __device__ __forceinline__ void load(const Rest<E>& r, int t0) {
    const int i = t0 + VEC * (threadIdx.x & 63);
#pragma unroll
    for (int k = 0; k < kBatch; ++k) p[k] = *reinterpret_cast<const Bits*>(r.p + from(i + k * TILE, r.V));
    if (r.s > 0.0) {
#pragma unroll
      for (int k = 0; k < kBatch; ++k) q[k] = *reinterpret_cast<const Bits*>(r.q + from(i + k * TILE, r.V));
    }
  }
  // The weights of tile k's tokens (its first one is `tile`) up to `end`.  All lanes call it.
  __device__ __forceinline__ void weights(const Rest<E>& r, int k, int tile, int end, double (&w)[VEC]) const {
    const int lane = threadIdx.x & 63, i = tile + VEC * lane;
#pragma unroll
    for (int j = 0; j < VEC; ++j) w[j] = prob(p[k].e[j]);
    if (r.s > 0.0) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) w[j] = fmax(fma(-r.s, static_cast<double>(prob(q[k].e[j])), w[j]), 0.0);
    }
    const int at = from(i, r.V);  // where the loaded ones begin
    if (tile + TILE > end) {
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (at + j < i || at + j >= end) w[j] = 0.0;
    }
    if (r.refused_of < 0) return;
    int x = r.mine;
    for (int c0 = r.refused_of + 1;;) {
      uint64_t hit = __builtin_amdgcn_ballot_w64(x >= tile && x < tile + TILE);
      while (hit != 0) {
        const int to = __builtin_amdgcn_readlane(x, __builtin_ctzll(hit)) - at;
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if (to == j) w[j] = 0.0;
        hit &= hit - 1;
      }
      c0 += 64;
      if (c0 >= r.n) return;
      x = c0 + lane < r.n && r.nodes->up[c0 + lane] == r.refused_of ? r.nodes->tok[c0 + lane] : -1;
    }
  }
};

// A wave's sum of the weights of tokens i0 .. i1 - 1; the next tiles are on their way while
// these are summed (eight at once instead, none ahead: 32 rows over 152064 tokens 24.0 us and 22.7, 128
// rows 32 and 35).
template <typename E, int VEC>
__device__ __forceinline__ double range_sum(const Rest<E>& r, int i0, int i1) {
  typedef Batch<E, VEC> B;
  double acc = 0.0;
  B next;
  next.load(r, i0);
  for (int t0 = i0; t0 < i1; t0 += kBatch * B::TILE) {
    const B now = next;
    if (t0 + kBatch * B::TILE < i1) next.load(r, t0 + kBatch * B::TILE);
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int tile = t0 + k * B::TILE;
      if (tile >= i1) break;
      double w[VEC];
      now.weights(r, k, tile, i1, w);
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc += w[j];
    }
  }
  return of_lane(wave_scan(acc), 63);
}

// The first token of i0 .. i1 - 1 (kBatch tiles at most) at which `before` plus the running sum passes t,
// else the last with a weight, else -1.  One wave.
template <typename E, int VEC>
__device__ __forceinline__ int find_token(const Rest<E>& r, int i0, int i1, double before, double t) {
  typedef Batch<E, VEC> B;
  int last = -1;
  B now;
  now.load(r, i0);
#pragma unroll
  for (int k = 0; k < kBatch; ++k) {
    const int tile = i0 + k * B::TILE, at = B::from(tile + VEC * (threadIdx.x & 63), r.V);
    if (tile >= i1) break;
    double w[VEC], own = 0.0;
    now.weights(r, k, tile, i1, w);
#pragma unroll
    for (int j = 0; j < VEC; ++j) own += w[j];
    const double upto = wave_scan(own);
    double c = before + (upto - own);
    int found = -1, any = -1;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      c += w[j];
      if (w[j] > 0.0) {
        any = at + j;
        if (found < 0 && c > t) found = at + j;
      }
    }
    const uint64_t hit = __builtin_amdgcn_ballot_w64(found >= 0), some = __builtin_amdgcn_ballot_w64(any >= 0);
    if (hit != 0) return __builtin_amdgcn_readlane(found, __builtin_ctzll(hit));
    if (some != 0) last = __builtin_amdgcn_readlane(any, 63 - __builtin_clzll(some));
    before += of_lane(upto, 63);
  }
  return last;
}

// Which of `many` sums (64 at most) the running sum from `before` passes t in, else the last one above
// zero; `before` becomes the running sum ahead of it.  All lanes call it.
__device__ __forceinline__ int narrow(const double* of, int many, double& before, double t) {
  const int lane = threadIdx.x & 63;
  const double own = lane < many ? of[lane] : 0.0, upto = wave_scan(own);
  const uint64_t some = __builtin_amdgcn_ballot_w64(own > 0.0), hit = __builtin_amdgcn_ballot_w64(own > 0.0 && before + upto > t);
  const int at = hit != 0 ? __builtin_ctzll(hit) : (some != 0 ? 63 - __builtin_clzll(some) : 0);
  before += of_lane(upto - own, at);
  return at;
}

// Where the sums of a row's parts are exchanged, and what the first launch gathers.
struct Shared {
  float2* probs;    // [T]: target's and draft's probability of the token, at the one that it follows
  uint64_t* slots;  // [B][kRounds][parts]
  int parts, part_len, polls;
};
constexpr int kRounds = 8;          // sums of a row that its workgroups share
constexpr int kMaxParts = 64;
constexpr uint64_t kMark = 1ull << 63;  // (no sum is negative: the sign says that it is there)

struct Row {
  int s, n;
};
__device__ __forceinline__ Row row_of(const fade_verify_args& a, int b) {
  const int T = static_cast<int>(a.T);
  int s = a.starts[b], e = a.starts[b + 1];
  s = s < 0 ? 0 : (s > T ? T : s);
  e = e < s ? s : (e > T ? T : e);
  return Row{s, e - s < kMaxNodes ? e - s : kMaxNodes};
}
__device__ __forceinline__ int parent_of(const fade_verify_args& a, const Row& r, int i) {
  const int up = i == 0 ? -1 : a.parents[r.s + i];
  return up >= 0 && up < i ? up : -1;
}
__device__ __forceinline__ int token_of(const fade_verify_args& a, const Row& r, int i) {
  const int64_t x = a.tok64 ? static_cast<const int64_t*>(a.tokens)[r.s + i] : static_cast<const int32_t*>(a.tokens)[r.s + i];
  return x >= 0 && x < a.V ? static_cast<int>(x) : -1;
}
template <typename E>
__device__ __forceinline__ float2 probs_of(const fade_verify_args& a, const Row& r, int up, int x) {
  if (up < 0 || x < 0) return make_float2(0.0f, 0.0f);
  const int64_t row = static_cast<int64_t>(r.s) + up;
  return make_float2(prob(static_cast<const E*>(a.target)[row * a.target_st + x]),
                     a.draft == nullptr ? 0.0f : prob(static_cast<const E*>(a.draft)[row * a.draft_st + x]));
}

template <typename E>
__global__ __launch_bounds__(256) void verify_gather_kernel(fade_verify_args a, Shared sh) {
  const int b = blockIdx.x;
  for (int i = threadIdx.x; i < kRounds * sh.parts; i += 256) sh.slots[static_cast<int64_t>(b) * kRounds * sh.parts + i] = 0;
  const Row r = row_of(a, b);
  for (int i = threadIdx.x; i < r.n; i += 256) sh.probs[r.s + i] = probs_of<E>(a, r, parent_of(a, r, i), token_of(a, r, i));
}

// A row's walk is made by all of its workgroups, each wave by itself, with the same results.
// Where a sum over the vocabulary is needed, each workgroup sums its part, stores it and
// reads the others' until they are there.  The wait is bounded: a workgroup that has polled
// `polls` times sums the missing parts itself, in the same order, to the same bits, so the
// kernel ends whatever part of it the chip runs at once.  From the sum number kRounds of a
// row on, its first workgroup goes on alone.  With one part nothing is exchanged.
// All sums, whatever they are for, are taken at one place of one loop: the kernel's code is
// fetched anew at each launch, and what it holds twice it fetches twice (with the sum's loop
// in six places 32 rows' trees took 37 us instead of 24).
template <typename E, int VEC, bool SHARED>
__global__ __launch_bounds__(kThreads) void verify_kernel(fade_verify_args a, Shared sh) {
  constexpr int TILE = 64 * VEC;
  __shared__ Nodes nodes;
  __shared__ double sums[kWaves], part_sums[kMaxParts];
  const int parts = SHARED ? sh.parts : 1;
  const int b = SHARED ? blockIdx.x / parts : blockIdx.x, part = SHARED ? blockIdx.x - b * parts : 0, V = static_cast<int>(a.V);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Row row = row_of(a, b);
  const int n = row.n;
  const int64_t out0 = static_cast<int64_t>(b) * a.max_path;
  auto put_token = [&](void* to, int64_t at, int64_t x) {
    if (a.tok64) static_cast<int64_t*>(to)[at] = x;
    else static_cast<int32_t*>(to)[at] = static_cast<int32_t>(x);
  };
  for (int i = threadIdx.x; i < n; i += kThreads) {
    // A token outside the vocabulary was drawn from nothing: it follows none, and so is never tried.  (Refused instead,
    // it would take draft's share from what is left, and the next token would not be the target's.)
    const int parent = parent_of(a, row, i), x = token_of(a, row, i), up = x < 0 ? -1 : parent;
    const float2 pq = SHARED ? sh.probs[row.s + i] : probs_of<E>(a, row, up, x);
    nodes.up[i] = static_cast<int16_t>(up);
    nodes.tok[i] = x;
    nodes.u[i] = a.uniforms[row.s + i];
    nodes.p[i] = pq.x;
    nodes.q[i] = pq.y;
  }
  const double final_u = a.final_u[b];
  __syncthreads();

  // token, the last child tried, tokens of the path, children refused here; q's share, the sum of what is left
  int cur = 0, last = 0, count = n > 0 ? 1 : 0, tried = 0;
  double share = 0.0, norm = 1.0;
  bool known = true;  // norm is of this share
  // 64 tokens at a time, one a lane: children come after their parents, so the walk never goes back
  int base = 0, up = -2, tok = -1;
  float p = 0.0f, q = 0.0f, u = 0.0f;
  auto look = [&]() {
    const int i = base + lane;
    up = -2;
    if (i < n) {
      up = nodes.up[i];
      tok = nodes.tok[i];
      p = nodes.p[i];
      q = nodes.q[i];
      u = nodes.u[i];
    }
  };
  look();
  if (n > 0 && part == 0 && threadIdx.x == 0) a.path[out0] = 0;
  auto put_next = [&](int x) {
    if (threadIdx.x != 0) return;
    if (count > 0) put_token(a.tokens_out, out0 + count - 1, x);
    put_token(a.next, b, x);
  };

  enum { kWalk, kEnd, kEndAgain, kNarrow };  // what the next sum is for
  int phase = kWalk, round = 0, item = 0, i0 = 0, i1 = 0;
  int polls = sh.polls;  // (of all rounds)
  double before = 0.0, t = 0.0;
  Rest<E> r;
  r.V = V;
  r.nodes = &nodes;
  r.n = n;
  for (;;) {
    if (phase == kWalk) {
      bool sum = false;
      while (count > 0 && count < a.max_path) {
        uint64_t who = __builtin_amdgcn_ballot_w64(up == cur && base + lane > last);  // the next children
        while (who == 0 && base + 64 < n) {
          base += 64;
          look();
          who = __builtin_amdgcn_ballot_w64(up == cur && base + lane > last);
        }
        if (who == 0) break;
        if (a.draft != nullptr && !known) {
          sum = true;
          break;
        }
        const int l = __builtin_ctzll(who), c = base + l, x = __builtin_amdgcn_readlane(tok, l);
        const double pc = of_lane(p, l), qc = of_lane(q, l);
        double left = pc, bound = of_lane(u, l) * norm;
        if (a.draft != nullptr) {
          left = fma(-share, qc, pc);
          bound *= qc;
        } else {
          // refused already?
          bool again = __builtin_amdgcn_ballot_w64(up == cur && tok == x && lane < l) != 0;
          for (int c0 = base - 64; c0 + 64 > cur && c0 >= 0; c0 -= 64)
            again |= __builtin_amdgcn_ballot_w64(nodes.up[c0 + lane] == cur && nodes.tok[c0 + lane] == x) != 0;
          if (again) left = 0.0;
        }
        last = c;
        if (left > 0.0 && bound < left) {
          if (part == 0 && threadIdx.x == 0) {
            a.path[out0 + count] = c;
            put_token(a.tokens_out, out0 + count - 1, x);
          }
          cur = c;
          ++count;
          tried = 0;
          share = 0.0;
          norm = 1.0;
          known = true;
        } else {
          ++tried;
          if (a.draft != nullptr) {
            share += norm;
            known = false;
          } else {
            norm -= left > 0.0 ? left : 0.0;
          }
        }
      }
      r.p = static_cast<const E*>(a.target) + (static_cast<int64_t>(row.s) + cur) * a.target_st;
      r.q = a.draft == nullptr ? nullptr : static_cast<const E*>(a.draft) + (static_cast<int64_t>(row.s) + cur) * a.draft_st;
      r.s = share;
      r.refused_of = -1;
      if (!sum) {
        phase = kEnd;
        if (part == 0) {
          for (int i = count + threadIdx.x; i < a.max_path; i += kThreads) {
            a.path[out0 + i] = -1;
            put_token(a.tokens_out, out0 + i, -1);
          }
          if (threadIdx.x == 0) a.counts[b] = count;
        }
        if (n == 0) {
          if (part == 0) put_next(-1);
          return;
        }
        if (a.draft == nullptr && tried > 0) {
          r.refused_of = cur;
          const int c = cur + 1 + lane;
          r.mine = c < n && nodes.up[c] == cur ? nodes.tok[c] : -1;
        }
      }
    }
    const bool shared = SHARED && round < kRounds;
    if (phase != kNarrow) {
      if (SHARED && !shared && part != 0) return;
      if (i1 == 0) item = shared ? part : 0;  // (else the next one of the sum that has begun)
      i0 = item * sh.part_len;
      i1 = i0 + sh.part_len < V ? i0 + sh.part_len : V;
    }

    // the sum, a share of the range in each wave
    const int seg = (i1 - i0 + kWaves * TILE - 1) / (kWaves * TILE) * TILE;
    {
      const int j0 = i0 + wave * seg, j1 = j0 + seg < i1 ? j0 + seg : i1;
      const double x = j0 < i1 ? range_sum<E, VEC>(r, j0, j1) : 0.0;
      __syncthreads();
      if (lane == 0) sums[wave] = x;
      __syncthreads();
    }

    if (phase != kNarrow) {
      const double own = of_lane(wave_scan(lane < kWaves ? sums[lane] : 0.0), 63);
      if (shared && item == part) {
        uint64_t* const slots = sh.slots + (static_cast<int64_t>(b) * kRounds + round) * parts;
        if (static_cast<int>(threadIdx.x) == part) {
          part_sums[part] = own;
          __hip_atomic_store(slots + part, __builtin_bit_cast(uint64_t, own) | kMark, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
        }
        if (static_cast<int>(threadIdx.x) < parts && static_cast<int>(threadIdx.x) != part) {
          uint64_t v;
          for (;;) {
            v = __hip_atomic_load(slots + threadIdx.x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
            if ((v & kMark) != 0 || --polls < 0) break;
            __builtin_amdgcn_s_sleep(1);
          }
          part_sums[threadIdx.x] = (v & kMark) != 0 ? __builtin_bit_cast(double, v & ~kMark) : -1.0;
        }
      } else if (threadIdx.x == 0) {
        part_sums[item] = own;
      }
      __syncthreads();
      // a part that is not there yet
      const double known_part = lane < parts ? part_sums[lane] : 0.0;
      const uint64_t missing = shared ? __builtin_amdgcn_ballot_w64(known_part < 0.0) : 0;
      if (shared ? missing != 0 : item + 1 < parts) {
        item = shared ? __builtin_ctzll(missing) : item + 1;
        __syncthreads();
        continue;
      }
      ++round;
      const double all = of_lane(wave_scan(known_part), 63);
      i1 = 0;
      if (phase == kWalk) {
        norm = all;
        known = true;
        continue;
      }
      if (!(all > 0.0)) {
        if (phase == kEndAgain) {
          if (part == 0) put_next(-1);
          return;
        }
        phase = kEndAgain;  // nothing is left: the token's probabilities themselves
        r.s = 0.0;
        r.refused_of = -1;
        continue;
      }
      // the part, the wave's share of it, a share of that, then the token
      t = final_u * all;
      const int owner = narrow(part_sums, parts, before, t);
      if (shared && owner != part) return;  // (its own workgroup goes on)
      phase = kNarrow;
      i0 = owner * sh.part_len;
      i1 = i0 + sh.part_len < V ? i0 + sh.part_len : V;
      if (owner != item) continue;
    }
    i0 += narrow(sums, kWaves, before, t) * seg;
    i1 = i0 + seg < i1 ? i0 + seg : i1;
    if (seg <= kBatch * TILE) break;  // (a wave reads as much at once)
    __syncthreads();
  }
  if (wave == 0) put_next(find_token<E, VEC>(r, i0, i1, before, t));
}

constexpr int kPolls = 256;        // about 1 us each: far beyond the wait of workgroups that run together
constexpr int kLeastPart = 4096;   // tokens of a part
constexpr int kLeastShared = 40000;  // tokens of a vocabulary that is shared out

// Tokens that a lane reads at once: 16 bytes, which a vocabulary of fewer does not have.
int vec_of(const fade_verify_args* a) {
  const int vec = a->dtype == FADE_DTYPE_F32 ? 4 : 8;
  return a->V < vec ? 1 : vec;
}

// The parts of a row's vocabulary: as many as give every CU a workgroup (one of this size finds a
// place there), if it has kLeastShared tokens.  Below, the exchange and the launch ahead of it
// cost more than one workgroup's pass (on the GPU, one row, a draft: 8000 tokens 6.6 us alone, shared
// 9.4; 32000 9.8 and 9.3; 64000 12.6 and 9.9; 152064 24 and 10.8; 32 rows' trees 11 and 16, 20 and
// 17.5, 28 and 17, 61 and 24), and the host's second launch and workspace 4 us.
Shared plan_of(const fade_verify_args* a, void* workspace) {
  const int tile = 64 * vec_of(a);
  int64_t parts = num_cus() / a->B;
  if (parts > cdiv(a->V, kLeastPart)) parts = cdiv(a->V, kLeastPart);
  if (parts > kMaxParts) parts = kMaxParts;
  if (parts < 1 || a->V < kLeastShared || a->T == 0) parts = 1;
  Shared sh;
  sh.part_len = static_cast<int>(cdiv(cdiv(a->V, parts), tile) * tile);
  sh.parts = static_cast<int>(cdiv(a->V, sh.part_len));
  sh.polls = a->polls < 0 ? 0 : (a->polls == 0 ? kPolls : a->polls);
  sh.slots = static_cast<uint64_t*>(workspace);
  sh.probs = reinterpret_cast<float2*>(sh.slots + a->B * kRounds * sh.parts);
  return sh;
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
  const Shared sh = plan_of(a, nullptr);
  *bytes = sh.parts < 2 ? 0 : (a->B * kRounds * sh.parts + a->T) * 8;
  return FADE_OK;
}

namespace {
template <typename E>
int launch(const fade_verify_args* a, const Shared& sh, hipStream_t st) {
  const unsigned B = static_cast<unsigned>(a->B);
  constexpr int VEC = 16 / sizeof(E);
  if (sh.parts < 2) {
    if (vec_of(a) == 1) hipLaunchKernelGGL((verify_kernel<E, 1, false>), dim3(B), dim3(kThreads), 0, st, *a, sh);
    else hipLaunchKernelGGL((verify_kernel<E, VEC, false>), dim3(B), dim3(kThreads), 0, st, *a, sh);
    return check_launch("fade_verify_drafts");
  }
  hipLaunchKernelGGL(verify_gather_kernel<E>, dim3(B), dim3(256), 0, st, *a, sh);
  const int rc = check_launch("fade_verify_drafts");
  if (rc) return rc;
  hipLaunchKernelGGL((verify_kernel<E, VEC, true>), dim3(B * sh.parts), dim3(kThreads), 0, st, *a, sh);
  return check_launch("fade_verify_drafts");
}
}  // namespace

FADE_API int fade_verify_drafts(const fade_verify_args* a, void* workspace, int64_t workspace_bytes, void* stream) {
  const int rc = check_args(a);
  if (rc) return rc;
  const Shared sh = plan_of(a, workspace);
  const int64_t need = sh.parts < 2 ? 0 : (a->B * kRounds * sh.parts + a->T) * 8;
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15)))
    return einval("fade_verify_drafts: needs a 16-byte aligned workspace of %lld bytes", (long long)need);
  hipStream_t st = as_stream(stream);
  if (a->dtype == FADE_DTYPE_F32) return launch<float>(a, sh, st);
  return a->dtype == FADE_DTYPE_BF16 ? launch<Bf16>(a, sh, st) : launch<uint16_t>(a, sh, st);
}
