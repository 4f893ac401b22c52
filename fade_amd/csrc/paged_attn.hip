// Attention of ragged chunks of new tokens over a paged 16-bit cache (gfx950).
//
// Row b brings n_b = starts[b + 1] - starts[b] new tokens (one in a decoding step,
// any number in a prompt's chunk) and holds L_b = lens[b] tokens, the new ones
// included, in pages of 64: token i lies in page table[b][i / 64].  Query i of the
// row sees keys 0 .. L_b - n_b + i (bottom-right causal) or all L_b:
//   o = sum_j p_j v_j / sum_j p_j,   p_j = exp2((q.k_j - m) * scale * log2 e)
// in one pass over the keys with the running maximum m and the sums in fp32.  A
// query that sees no key gets zeros.
//
// The G = Hq / Hkv query heads of a kv head times the n_b queries are the matrix
// rows of (row b, kv head): row r is query r / G, head r % G, so any G and any
// chunk length fill the same tiles and each key is read once per tile of rows.
//
// Work is cut on the device, from the lengths the host does not know.  A tile is M
// matrix rows of a (row b, kv head); its cost is the keys that it reads and a
// constant for its start and end.  The tiles of all rows lie one after the other on
// a line, and every workgroup of a kv head takes an equal piece of it, whatever the
// rows' lengths are: the end of one tile, whole tiles, the beginning of another (a
// border close to a tile's own is moved there, where a cut costs more than that).  A
// wave finds its place by a sum over the rows' costs (one load per lane for 64
// rows).  Whole tiles are written out; a tile cut by a piece's border leaves
// unnormalized fp32 sums, at most two per workgroup, which a second launch joins in
// the order of the keys, so results do not depend on timing.
#include <math.h>

#include "fade_common.h"
#include "lds_dma.h"

namespace fade {
namespace paged {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
typedef __attribute__((address_space(3))) uint8_t lds_u8;
typedef __attribute__((address_space(4))) int32_t const_i32;

constexpr int kThreads = 256;
constexpr int kPage = 64;
constexpr int kRows = 16;  // matrix rows of an item of the few-row kernel
constexpr float kNegBig = -3.402823466e38f;  // no score is lower

template <int V>
struct Int {
  static constexpr int value = V;
};

enum { kAll = 0, kFew = 1, kMany = 2 };

struct Params {
  int64_t B, T, ppr, n_pages;
  int Hq, Hkv, G, D;
  const uint16_t* q;
  int64_t q_st, q_sh;
  uint16_t* out;
  int64_t o_st, o_sh;
  const uint16_t* kp;
  const uint16_t* vp;
  const int32_t* table;
  const int32_t* lens;
  const int32_t* starts;
  float scale_log2;
  int causal;
  int zero_tail;
  // the cut of one kernel's work
  int rows_of;     // kAll, or the rows of the batch whose matrix rows fit one tile of 16 (kFew) or do not (kMany)
  int lm;          // log2 of the matrix rows of a tile
  int per_tile;    // queries that a tile touches at most
  int start_cost;  // of a tile, in keys
  int pieces;      // workgroups per kv head
  float per_piece; // a little over 1 / pieces
  int least;       // fewest keys of a piece
  int snap;        // a border this near to a tile's is moved there
  float* part_o;   // [workgroup][2][M][D]: a tile's end (0), a tile's beginning (1)
  float2* part_ml; // [workgroup][2][M]: maximum (log2 units, less what its kernel holds probabilities larger by), sum
  int4* cuts;      // [workgroup]: the tile that begins in its piece and ends in another: first new token, its
                   // first matrix row, matrix rows of the row, parts (0: none)
};

// A tile (wave-uniform).
struct Tile {
  int b, q0, n, len;   // row, its first new token, new tokens, tokens
  int tile;            // of the row's tiles
  uint64_t at, cost;   // its place on the line
};
// Where the search of the next tile starts: rows b0 .., their place on the line.
struct Place {
  int b0;
  uint64_t before;
};

// A row's new tokens and length from device data, kept inside the tensors.
__device__ __forceinline__ void row_counts(const Params& p, int b, int& q0, int& n, int& len) {
  const int T = static_cast<int>(p.T);
  int s = p.starts[b], e = p.starts[b + 1];
  s = s < 0 ? 0 : (s > T ? T : s);
  e = e < s ? s : (e > T ? T : e);
  const int cap = static_cast<int>(p.ppr) * kPage;
  const int l = p.lens[b];
  q0 = s;
  n = e - s;
  len = l < 0 ? 0 : (l > cap ? cap : l);
}
__device__ __forceinline__ uint32_t tiles_of(const Params& p, int n) {
  const uint32_t rows = static_cast<uint32_t>(n) * static_cast<uint32_t>(p.G);
  if (p.rows_of != kAll && (rows <= kRows) != (p.rows_of == kFew)) return 0u;
  return (rows + (1u << p.lm) - 1u) >> p.lm;
}
// Cost of a row's first t tiles: tile i reads at most base + step (i + 1) keys.
__device__ __forceinline__ uint64_t cost_of(const Params& p, int n, int len, uint64_t t) {
  const uint64_t step = p.causal ? p.per_tile : 0;
  const int base = p.causal ? (len > n ? len - n : 0) : len;
  return t * static_cast<uint64_t>(base + p.start_cost) + step * (t * (t + 1) / 2);
}

// Inclusive sums over the wave's lanes: shifts within rows of 16 lanes, then each
// row's last lane to the next row (DPP: no LDS round trips).
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t scan_step(uint64_t v) {
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xF, true);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(v >> 32), CTRL, ROWS, 0xF, true);
  return v + ((static_cast<uint64_t>(hi) << 32) | lo);
}
__device__ __forceinline__ uint64_t wave_scan(uint64_t v) {
  v = scan_step<0x111, 0xF>(v);  // row_shr 1, 2, 4, 8
  v = scan_step<0x112, 0xF>(v);
  v = scan_step<0x114, 0xF>(v);
  v = scan_step<0x118, 0xF>(v);
  v = scan_step<0x142, 0xA>(v);  // row_bcast 15 to rows 1 and 3
  return scan_step<0x143, 0xC>(v);  // row_bcast 31 to rows 2 and 3
}
__device__ __forceinline__ uint64_t lane_of(uint64_t v, int l) {
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(v), l), hi = __builtin_amdgcn_readlane(static_cast<int>(v >> 32), l);
  return (static_cast<uint64_t>(hi) << 32) | lo;
}
__device__ __forceinline__ uint64_t uniform(uint64_t v) { return lane_of(v, 0); }

// A lane's row of the 64 that a wave looks at.
struct Row {
  int q0, n, len;
  uint64_t cost;
};
__device__ __forceinline__ Row row_of(const Params& p, int b) {
  Row r{0, 0, 0, 0};
  if (b < p.B) {
    row_counts(p, b, r.q0, r.n, r.len);
    r.cost = cost_of(p, r.n, r.len, tiles_of(p, r.n));
  }
  return r;
}

// Length of the line, and of a piece of it; `first`: the lane's row of rows 0 .. 63.
// All lanes of the wave call it.
__device__ __forceinline__ void line_of(const Params& p, uint64_t& all, uint64_t& piece, Row& first) {
  const int B = static_cast<int>(p.B), lane = threadIdx.x & 63;
  first = row_of(p, lane);
  uint64_t work = first.cost;
  for (int b = lane + 64; b < B; b += 64) work += row_of(p, b).cost;
  all = lane_of(wave_scan(work), 63);
  // (the factor keeps piece * pieces at or above the line's length despite the roundings)
  piece = uniform(static_cast<uint64_t>(static_cast<float>(all) * p.per_piece) + 1);
  if (piece < static_cast<uint64_t>(p.least)) piece = p.least;
}

// The tile at place x of the line, at or after `from`'s rows; false past the end.
__device__ __forceinline__ bool find_tile(const Params& p, uint64_t x, const Row& first, Place& from, Tile& w) {
  const int lane = threadIdx.x & 63, B = static_cast<int>(p.B);
  for (int b0 = from.b0; b0 < B; b0 += 64) {
    const Row r = b0 == 0 ? first : row_of(p, b0 + lane);
    const uint64_t to = from.before + wave_scan(r.cost);
    const uint64_t who = __builtin_amdgcn_ballot_w64(x < to && x >= to - r.cost);
    if (who != 0) {
      const int l = __builtin_ctzll(who);
      w.b = b0 + l;
      w.q0 = __builtin_amdgcn_readlane(r.q0, l);
      w.n = __builtin_amdgcn_readlane(r.n, l);
      w.len = __builtin_amdgcn_readlane(r.len, l);
      const uint64_t row_at = lane_of(to - r.cost, l), off = x - row_at;
      const int tiles = __builtin_amdgcn_readfirstlane(static_cast<int>(tiles_of(p, w.n)));
      if (tiles == 1) {
        w.tile = 0;
        w.at = row_at;
        w.cost = lane_of(r.cost, l);
        return true;
      }
      // the tile: cost_of(tile) <= off < cost_of(tile + 1), by its real solution and a step to either side
      const double step = p.causal ? p.per_tile : 0;
      const double a = (p.causal ? (w.len > w.n ? w.len - w.n : 0) : w.len) + p.start_cost + 0.5 * step;
      const double guess = step > 0.0 ? 2.0 * static_cast<double>(off) / (a + sqrt(a * a + 2.0 * step * static_cast<double>(off)))
                                      : static_cast<double>(off) / a;
      int t = __builtin_amdgcn_readfirstlane(static_cast<int>(guess));
      t = t < 0 ? 0 : (t >= tiles ? tiles - 1 : t);
      while (t > 0 && cost_of(p, w.n, w.len, t) > off) --t;
      while (t + 1 < tiles && cost_of(p, w.n, w.len, t + 1) <= off) ++t;
      w.tile = t;
      const uint64_t c0 = cost_of(p, w.n, w.len, t);
      w.at = row_at + c0;
      w.cost = cost_of(p, w.n, w.len, t + 1) - c0;
      return true;
    }
    from.b0 = b0 + 64;
    from.before = lane_of(to, 63);
  }
  return false;
}

// One workgroup's walk over its piece of the line.
struct Walk {
  uint64_t x, end, piece, snap;
  Place from;
  Row lane_row;     // the lane's row of rows 0 .. 63
  int tokens;       // new tokens of all rows (p.zero_tail)
  Tile w;
  int lo, hi;       // the keys of the tile in this piece: lo to hi (of steps of `grain` keys)
  bool first, last; // the piece holds the tile's beginning, its end
};
__device__ __forceinline__ bool walk_start(const Params& p, int piece_index, Walk& k) {
  uint64_t all, piece;
  k.tokens = p.zero_tail ? p.starts[p.B] : 0;
  line_of(p, all, piece, k.lane_row);
  k.x = piece * static_cast<uint64_t>(piece_index);
  k.end = k.x + piece < all ? k.x + piece : all;
  k.from = Place{0, 0};
  k.piece = piece;
  k.snap = piece / 3 < static_cast<uint64_t>(p.snap) ? piece / 3 : p.snap;
  k.first = k.last = false;
  return k.x < k.end;
}
// Where the border x, inside the tile from `at` to `end`, comes to lie: at the
// nearer end of the tile, if that is near.
__device__ __forceinline__ uint64_t snapped(const Walk& k, uint64_t x, uint64_t at, uint64_t end) {
  const uint64_t d0 = x - at, d1 = end - x;
  if ((d0 < d1 ? d0 : d1) > k.snap) return x;
  return d0 < d1 ? at : end;
}
// The next tile of the piece; `grain`: keys that are not divided.
__device__ __forceinline__ bool walk_next(const Params& p, int grain, Walk& k) {
  Tile t;
  uint64_t tile_end;
  do {
    if (k.x >= k.end || !find_tile(p, k.x, k.lane_row, k.from, t)) return false;
    tile_end = t.at + t.cost;
    if (tile_end <= k.x) return false;  // (counts that contradict each other)
    if (k.x != t.at) k.x = snapped(k, k.x, t.at, tile_end);  // the piece's begin
  } while (k.x == tile_end);
  uint64_t end = k.end;
  if (end < tile_end) {
    end = snapped(k, end, t.at, tile_end);
    if (end == t.at) return false;
  }
  k.w = t;
  const Tile& w = k.w;
  const int rows = w.n * p.G, last_row = ((w.tile + 1) << p.lm) < rows ? ((w.tile + 1) << p.lm) : rows;
  int seen = p.causal ? w.len - w.n + (last_row - 1) / p.G + 1 : w.len;  // keys that the tile's last row sees
  seen = seen < 0 ? 0 : seen;
  k.first = k.x == w.at;
  k.last = tile_end <= end;
  const int a = static_cast<int>(k.x - w.at) / grain * grain, e = static_cast<int>(k.end - w.at) / grain * grain;
  k.lo = a < seen ? a : seen;
  k.hi = k.last || e > seen ? seen : e;
  k.lo = __builtin_amdgcn_readfirstlane(k.lo);
  k.hi = __builtin_amdgcn_readfirstlane(k.hi);
  k.x = tile_end;
  return true;
}

// Rows of q past the last sequence: zeros, where the caller asked for them.
__device__ __forceinline__ void zero_tail(const Params& p, int end, int64_t block, int64_t blocks, int kvh) {
  end = end < 0 ? 0 : end;
  const int G = p.G;
  for (int64_t t = end + block; t < p.T; t += blocks)
    for (int i = threadIdx.x; i < G * p.D; i += blockDim.x)
      p.out[t * p.o_st + (static_cast<int64_t>(kvh) * G + i / p.D) * p.o_sh + i % p.D] = 0;
}

// The end of a workgroup.  What the second launch has to join: the piece's last
// tile, if it begins here and ends elsewhere.
__device__ __forceinline__ void finish(const Params& p, const Walk& k, bool any) {
  if (p.zero_tail) zero_tail(p, k.tokens, blockIdx.x / p.Hkv, gridDim.x / p.Hkv, blockIdx.x % p.Hkv);
  if (p.pieces < 2 || threadIdx.x != 0) return;
  int parts = 0;
  if (any && k.first && !k.last) {
    const uint64_t rest = k.w.at + k.w.cost - k.end;  // > 0: in the next pieces
    parts = static_cast<int>(static_cast<double>(rest) / static_cast<double>(k.piece));  // (a whole number or two off)
    if (parts > 0) --parts;
    while (k.piece * static_cast<uint64_t>(parts) < rest && parts < p.pieces) ++parts;
    // (the last border in the tile may be the tile's own)
    if (parts < 2 || rest - k.piece * static_cast<uint64_t>(parts - 1) > k.snap) ++parts;
  }
  p.cuts[blockIdx.x] = make_int4(k.w.q0, k.w.tile << p.lm, k.w.n * p.G, parts);
}

template <bool BF>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <bool BF>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (BF) return pack_bf16(a, b);
  else return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), f16x2));
}

// Values that are no numbers.  A probability of zero does not hide an infinity or a
// NaN from a product, so one of a token that a row does not see would reach it.  A
// tile whose sums hold a NaN at the end of a piece is therefore walked once more:
// each step's values are looked through, the rows add what is no number of the keys
// that they see by themselves, and the products find zeros in their places.
template <bool BF>
struct Odd {
  static constexpr uint32_t kExp = BF ? 0x7F80 : 0x7C00;
  // whether one of the N KB at `at` (LDS) is an infinity or a NaN
  template <int N>
  static __device__ __forceinline__ bool any(const uint8_t* at, int lane) {
    u16x8 top = {};
#pragma unroll 2
    for (int i = 0; i < N; ++i)
      top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x8, *reinterpret_cast<const u32x4*>(at + 1024 * i + 16 * lane) & 0x7FFF7FFFu));
    const auto t2 = __builtin_elementwise_max(__builtin_elementwise_max(top.s01, top.s23), __builtin_elementwise_max(top.s45, top.s67));
    return __builtin_amdgcn_ballot_w64(t2.x >= kExp || t2.y >= kExp) != 0;
  }
  static __device__ __forceinline__ uint32_t finite(uint32_t v) {
    if ((v & kExp) == kExp) v &= 0xFFFF0000u;
    if ((v >> 16 & kExp) == kExp) v &= 0xFFFFu;
    return v;
  }
  // zeros in their places, in the BYTES bytes at `at` (LDS), by THREADS threads
  template <int BYTES, int THREADS>
  static __device__ __forceinline__ void clear(uint8_t* at) {
#pragma unroll 1
    for (int i = 4 * threadIdx.x; i < BYTES; i += 4 * THREADS) *reinterpret_cast<uint32_t*>(at + i) = finite(*reinterpret_cast<const uint32_t*>(at + i));
  }
  // x += what of v is no number
  static __device__ __forceinline__ float added(float x, uint32_t v) { return (v & kExp) == kExp ? x + w2f<BF>(static_cast<uint16_t>(v)) : x; }
};

// ---- few rows: tiles of 16 matrix rows, one wave per workgroup ----
//
// The wave walks its piece in steps of 32 keys.  K and V rows go from the page
// straight to LDS (no register holds them, no barrier is needed), two steps deep:
// the next step's loads fly while this one is computed.  Four such waves per CU
// (head_dim 128) keep 64 KB of loads in flight, and one's start or end runs beside
// the others' loads.  Bound by HBM: 16 rows over 8000 keys each (32 heads, 8 kv
// heads of 128) 103 us, 5.2 TB/s, as a large copy has; 64 rows of 10 to 9000 keys
// 149 us.  Eight waves per CU 111 us, sixteen 120; three steps deep no faster.  A
// single row of few keys is bound by latency: 6.5 us and 3.5 for the join.
//   S^T = K Q^T   16x16x32 MFMAs, A = 16 keys x 32 channels, B = Q^T (registers):
//                 lane (n, g) holds query row n, keys 4 g + i of the 16
//   O^T += V^T P^T  A = V^T by transposing LDS reads (4 keys x 16 channels each),
//                 B = P^T straight from S^T's registers: k slot (g, j) is key
//                 4 g + j of the first 16 keys (j < 4), 4 g + j - 4 of the second
// so the running maximum, the sum and the rescaling are lane-local; P is multiplied
// as a 16-bit head plus a 16-bit rest (P to 2^-16 or better): the matrix cores are
// idle here, and rounding P alone would cost as much accuracy as rounding the output.
// fp16 holds nothing finer than 2^-24, and where one key takes the weight (a sink)
// the output is what many light ones add up to: P and its sum are held 2^15 times
// larger there, P to 2^-40 of the largest.
// 16-byte unit u of LDS row r lies at unit u ^ (2 (r & 7)) (mod the row), which the
// loads' source addresses bring about: without it the 16 rows that a transposing
// read touches would share their banks.
template <int DP>
struct Few {
  static constexpr int kKeys = 32;                 // keys per step
  static constexpr int kUnits = DP / 8;            // 16-byte units per row
  static constexpr int kTensor = kKeys * DP * 2;   // bytes of a step's K or V
  static constexpr int kStage = 2 * kTensor;
  static constexpr int kLoads = kStage / 1024;     // direct loads per step
  static constexpr int kStages = 2;                // (the waits below count one step ahead)
  static_assert(kLoads < 64, "vmcnt counts to 63");
  static constexpr int kQBytes = kRows * DP * 2;
  static constexpr int kLds = kStages * kStage + kQBytes;
  static constexpr int kSwizzle = kUnits - 1;
  static constexpr float kHeld = 15.0f;            // log2 of the factor on fp16 probabilities, which are 1 at most
};

template <int DP>
__device__ __forceinline__ int few_unit(int row, int u) {
  return u ^ ((2 * row) & Few<DP>::kSwizzle);
}

template <int DP, bool BF>
__global__ __launch_bounds__(64) void paged_few_kernel(Params p) {
  typedef Few<DP> F;
  constexpr int NKS = DP / 32, NCB = DP / 16;
  const int kvh = blockIdx.x % p.Hkv, index = blockIdx.x / p.Hkv;
  const int lane = threadIdx.x, n16 = lane & 15, g = lane >> 4;
  Walk k;
  k.w = Tile{};
  if (!walk_start(p, index, k)) {
    finish(p, k, false);
    return;
  }
  const int D = p.D;

  __shared__ __attribute__((aligned(16))) uint8_t lds[F::kLds];
  const uint32_t base = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_u8*)lds)));
  if (D < DP) {  // units past the head_dim are never loaded: zeros
    for (int i = 16 * lane; i < F::kStages * F::kStage; i += 1024) *reinterpret_cast<u32x4*>(lds + i) = u32x4{0, 0, 0, 0};
    __builtin_amdgcn_s_waitcnt(kLgkm0);
  }
  while (walk_next(p, F::kKeys, k)) {
    const Tile& w = k.w;
    const int all = w.n * p.G, r = w.tile * kRows + n16;  // this lane's matrix row: its query, head and visible keys
    const bool live = r < all;
    const int qi = live ? r / p.G : 0, hd = kvh * p.G + (live ? r - qi * p.G : 0);
    auto limit = [&](int i) {
      const int x = p.causal ? w.len - w.n + i + 1 : w.len;
      return x < 0 ? 0 : x;
    };
    const int lim = live ? limit(qi) : 0;
    const int seen_by_all = __builtin_amdgcn_readfirstlane(limit(w.tile * kRows / p.G));  // the tile's first row sees the fewest

    const const_i32* trow = (const const_i32*)(uintptr_t)(p.table + w.b * p.ppr);  // (scalar loads: vmcnt counts the steps' alone)
    auto issue = [&](int key, int id, int buf) {
      id = id < 0 || id >= p.n_pages ? 0 : id;
      const int64_t at = ((static_cast<int64_t>(id) * p.Hkv + kvh) * kPage + key % kPage) * D;
      const uint32_t to = base + buf * F::kStage;
#pragma unroll
      for (int i = 0; i < F::kLoads / 2; ++i) {
        const int pos = 64 * i + lane, row = pos / F::kUnits;
        const int u = few_unit<DP>(row, pos % F::kUnits);
        if (DP == D || 8 * u < D) {
          lds_dma16(p.kp + at + row * D + 8 * u, to + 1024 * i);
          lds_dma16(p.vp + at + row * D + 8 * u, to + F::kTensor + 1024 * i);
        }
      }
    };
    // the query's rows to LDS ahead of the keys (16-byte unit i of the tile's 16 rows: row i / kUnits)
    const uint32_t qlds = base + F::kStages * F::kStage;
#pragma unroll
    for (int i = 0; i < F::kQBytes / 1024 + (F::kQBytes % 1024 != 0); ++i) {
      const int pos = 64 * i + lane, row = pos / F::kUnits, u = pos % F::kUnits;
      const int rr = w.tile * kRows + row, ri = rr < all ? rr : all - 1, rq = ri / p.G;
      if (DP == D || 8 * u < D)
        lds_dma16(p.q + static_cast<int64_t>(w.q0 + rq) * p.q_st + static_cast<int64_t>(kvh * p.G + ri - rq * p.G) * p.q_sh + 8 * u, qlds + 1024 * i);
    }
    f32x4 acc[NCB];
    float m, l;  // of row n16 (l: over this lane's keys)
    for (bool again = false;; again = true) {
      int key = k.lo, ahead = k.lo, next = 0;  // ahead: the first key not asked for
#pragma unroll
      for (int i = 0; i < F::kStages - 1; ++i)
        if (ahead < k.hi) {
          issue(ahead, __builtin_amdgcn_readfirstlane(trow[ahead / kPage]), i);
          ahead += F::kKeys;
        }
      if (ahead < k.hi) next = trow[ahead / kPage];
      u32x4 qf[NKS];
      {
        // the query's loads are done when no more than the steps' are in flight
        if (ahead > key) __builtin_amdgcn_s_waitcnt(vmcnt_imm(F::kLoads));
        else __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
        asm volatile("" ::: "memory");
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) {
          const int c = 32 * ks + 8 * g;
          const u32x4 x = *reinterpret_cast<const u32x4*>(lds + F::kStages * F::kStage + 2 * (n16 * DP + c));
          qf[ks] = DP == D || c < D ? x : u32x4{0, 0, 0, 0};
        }
      }
#pragma unroll
      for (int cb = 0; cb < NCB; ++cb) acc[cb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      m = -INFINITY;
      l = 0.0f;
      for (int t = 0; key < k.hi; key += F::kKeys, t = t + 1 == F::kStages ? 0 : t + 1) {
        if (ahead < k.hi) {
          issue(ahead, __builtin_amdgcn_readfirstlane(next), t == 0 ? F::kStages - 1 : t - 1);
          ahead += F::kKeys;
          if (ahead < k.hi) next = trow[ahead / kPage];
          __builtin_amdgcn_s_waitcnt(vmcnt_imm(F::kLoads));
        } else {
          __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
        }
        asm volatile("" ::: "memory");
        uint8_t* const kt = lds + t * F::kStage;
        uint8_t* const vt = kt + F::kTensor;
        const int cnt = w.len - key;  // rows from here on hold no token of the row: whatever stands there must not count
        if (cnt < F::kKeys) {
          for (int i = lane; i < (F::kKeys - cnt) * F::kUnits; i += 64)
            *reinterpret_cast<u32x4*>(vt + 16 * (cnt * F::kUnits + i)) = u32x4{0, 0, 0, 0};
        }
        f32x4 s[2];
#pragma unroll
        for (int kt16 = 0; kt16 < 2; ++kt16) {
          s[kt16] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
          const int row = 16 * kt16 + n16;
#pragma unroll
          for (int ks = 0; ks < NKS; ++ks) {
            const u32x4 a = *reinterpret_cast<const u32x4*>(kt + row * DP * 2 + 16 * few_unit<DP>(row, 4 * ks + g));
            s[kt16] = mfma16<BF>(a, qf[ks], s[kt16]);
          }
        }
        float x[8], tm = -INFINITY;
        const bool whole = key + F::kKeys <= seen_by_all;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[i] = s[i >> 2][i & 3] * p.scale_log2;
          if (!whole && key + 16 * (i >> 2) + 4 * g + (i & 3) >= lim) x[i] = -INFINITY;
          tm = fmaxf(tm, x[i]);
        }
        tm = fmaxf(tm, __shfl_xor(tm, 16, 64));
        tm = fmaxf(tm, __shfl_xor(tm, 32, 64));
        const float mn = fmaxf(m, tm);
        const float ms = mn == -INFINITY ? 0.0f : mn;
        float alpha = __builtin_amdgcn_exp2f(m - ms);
        m = mn;
        float ps = 0.0f;
        u32x4 ph, pl;
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          float da = x[i] - ms, db = x[i + 1] - ms;
          if constexpr (!BF) {  // (2^15 times, not added to ms: its rounding there would differ from step to step)
            da += F::kHeld;
            db += F::kHeld;
          }
          const float a = __builtin_amdgcn_exp2f(da), b = __builtin_amdgcn_exp2f(db);
          ps += a + b;
          const uint32_t h = pack2<BF>(a, b);
          ph[i / 2] = h;
          pl[i / 2] = pack2<BF>(a - w2f<BF>(static_cast<uint16_t>(h)), b - w2f<BF>(static_cast<uint16_t>(h >> 16)));
        }
        l = l * alpha + ps;
        auto value_frag = [&](int cb) {
          // lane (n, g) points at key 4 g + n / 4 (+ 16), channels 16 cb + 4 (n % 4) .. + 3
          const int row = 4 * g + (n16 >> 2), u = 2 * cb + ((n16 >> 1) & 1);
          const uint8_t* at = vt + row * DP * 2 + 16 * few_unit<DP>(row, u) + 8 * (n16 & 1);
          const i16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_i16x4*>((lds_u8*)const_cast<uint8_t*>(at)));
          const i16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              reinterpret_cast<lds_i16x4*>((lds_u8*)const_cast<uint8_t*>(at + 16 * DP * 2)));  // (row + 16: the same swizzle)
          const u32x2 w0 = __builtin_bit_cast(u32x2, v0), w1 = __builtin_bit_cast(u32x2, v1);
          return u32x4{w0.x, w0.y, w1.x, w1.y};
        };
        if (again && Odd<BF>::template any<F::kTensor / 1024>(vt, lane)) {
#pragma unroll
          for (int cb = 0; cb < NCB; ++cb)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[cb][i] *= alpha;
#pragma unroll 1
          for (int j = 0; j < F::kKeys && key + j < lim; ++j)
#pragma unroll
            for (int cb = 0; cb < NCB; ++cb) {  // channels 16 cb + 4 g .. + 3
              const u32x2 v = *reinterpret_cast<const u32x2*>(vt + j * DP * 2 + 16 * few_unit<DP>(j, 2 * cb + (g >> 1)) + 8 * (g & 1));
#pragma unroll
              for (int i = 0; i < 4; ++i) acc[cb][i] = Odd<BF>::added(acc[cb][i], v[i >> 1] >> (16 * (i & 1)));
            }
          Odd<BF>::template clear<F::kTensor, 64>(vt);
          asm volatile("" ::: "memory");
          alpha = 1.0f;
        }
#pragma unroll
        for (int cb = 0; cb < NCB; ++cb) {
          const u32x4 a = value_frag(cb);
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[cb][i] *= alpha;
          acc[cb] = mfma16<BF>(a, ph, acc[cb]);
          acc[cb] = mfma16<BF>(a, pl, acc[cb]);
        }
      }
      bool nan = false;
#pragma unroll
      for (int cb = 0; cb < NCB; ++cb)
#pragma unroll
        for (int i = 0; i < 4; ++i) nan |= acc[cb][i] != acc[cb][i];
      if (again || __builtin_amdgcn_ballot_w64(nan) == 0) break;
    }
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    // ---- lane (n, g): row n, channels 16 cb + 4 g .. + 3 ----
    if (!live) continue;
    if (k.first && k.last) {
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // no visible key: zeros
      uint16_t* dst = p.out + static_cast<int64_t>(w.q0 + qi) * p.o_st + static_cast<int64_t>(hd) * p.o_sh;
#pragma unroll
      for (int cb = 0; cb < NCB; ++cb) {
        const int c = 16 * cb + 4 * g;
        if (c < D)
          *reinterpret_cast<u32x2*>(dst + c) = u32x2{pack2<BF>(acc[cb][0] * inv, acc[cb][1] * inv), pack2<BF>(acc[cb][2] * inv, acc[cb][3] * inv)};
      }
    } else {
      const int64_t pr = (static_cast<int64_t>(blockIdx.x) * 2 + (k.first ? 1 : 0)) * kRows + n16;
      if (g == 0) p.part_ml[pr] = make_float2(m, l);
#pragma unroll
      for (int cb = 0; cb < NCB; ++cb) {
        const int c = 16 * cb + 4 * g;
        if (c < D) *reinterpret_cast<f32x4*>(p.part_o + pr * D + c) = acc[cb];
      }
    }
  }
  finish(p, k, true);
}

// ---- many rows: tiles of 32 NW matrix rows, the keys shared through LDS ----
//
// NW waves of 32 matrix rows each walk the tile's keys in steps of KT.  A step's K
// and V go straight to LDS, NST steps' buffers in a ring, every wave loading its
// share; one barrier per step.
//   S^T = K Q^T   32x32x16 MFMAs, A = 32 keys x 16 channels, B = Q^T (registers):
//                 lane (n, h) holds matrix row n, register i key 8 (i / 4) + 4 h + i % 4
//   O^T += V^T P^T  A = V^T by transposing LDS reads, B = P^T straight from S^T's
//                 registers: k slot (h, j) of step s is key 16 s + 4 h + j (j < 4),
//                 16 s + 8 + 4 h + j - 4
// so a row's maximum, sum and rescaling are lane-local.  The running maximum moves
// only where a probability passes 2^8 (fp16: 2^6; found on the 16-bit probabilities,
// two per operation; the exact maximum is taken there alone), so most steps need
// neither a maximum of the scores nor an exchange between lanes nor a rescaling.  P is
// rounded to 16 bits (as the output is; the sum takes the same rounded values): a
// second product for its rest would cost half the matrix work again.  fp16
// probabilities are held 2^9 times larger, so that a key 2^23 times lighter than the
// heaviest one still counts with all 11 bits (2^34 times lighter: not at all); eight
// chunks of 128 to 2048 tokens 505 us, not held larger 501, 2^11 times 515, 2^12 times
// 525 (they pass their bound, and are rescaled, more often).
//
// Eight chunks of 128 to 2048 tokens over up to 11K keys (32 heads, 8 kv heads of
// 128): 500 to 670 us by the drawn lengths and the card's state, 1040 TFLOP/s of
// visible keys at 565.  What bounds it is the power
// that the card has: its matrix instructions alone reach 1370 TFLOP/s on random
// numbers (2200 on constant ones), with this kernel's LDS reads and exponentials
// beside them 1296, with its loads and barriers 1090.  Measured without gain: scores
// of the next step beside this step's exponentials, a barrier per two steps, 2 to 4
// buffers, 64 rows per wave.  256-row tiles: 128-row ones (4 waves, two workgroups a
// CU) 700 us against 657 then; steps of 32 keys at head_dim over 128, where the
// accumulators and the query leave registers for one block of scores.
// LDS rows are DP channels, 16-byte units exchanged so that the eight (16) rows
// that a read of K touches and the four that a transposing read of V touches lie
// in different banks.
template <int DP>
__device__ __forceinline__ int wide_k_unit(int row, int u) {
  if constexpr (DP == 64) return u ^ ((row >> 1) & 7);
  else return u ^ (row & 15);
}
template <int DP>
__device__ __forceinline__ int wide_v_unit(int row, int u) {
  if constexpr (DP == 64) return u ^ (4 * ((row >> 1) & 1));
  else return u ^ (4 * (row & 3));
}
__device__ __forceinline__ u32x4 lds_read16(uint32_t at) {
  return *reinterpret_cast<const __attribute__((address_space(3))) u32x4*>(at);
}
__device__ __forceinline__ u32x2 lds_read_tr(uint32_t at) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_i16x4*>(at)));
}
template <bool BF>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <int DP, int NW, int KT, int NST, bool BF>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(2, 2))) void paged_wide_kernel(Params p) {
  constexpr int M = 32 * NW;
  constexpr int NKS = DP / 16, NCB = DP / 32, UNITS = DP / 8;
  constexpr int TENSOR = KT * DP * 2, STAGE = 2 * TENSOR, NKB = KT / 32;
  constexpr int LPW = TENSOR / 1024 / NW;  // direct loads of K, and of V, per wave and page
  static_assert(TENSOR % (1024 * NW) == 0, "a page is shared out evenly");
  const int kvh = blockIdx.x % p.Hkv, index = blockIdx.x / p.Hkv;
  const int lane = threadIdx.x & 63, n32 = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Walk k;
  k.w = Tile{};
  if (!walk_start(p, index, k)) {
    finish(p, k, false);
    return;
  }
  const int D = p.D;

  __shared__ __attribute__((aligned(256))) uint8_t lds[NST * STAGE];
  __shared__ int any_nan;
  const uint32_t base = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_u8*)lds)));
  if (D < DP) {  // units past the head_dim are never loaded: zeros
    for (int i = 16 * threadIdx.x; i < NST * STAGE; i += 1024 * NW) *reinterpret_cast<u32x4*>(lds + i) = u32x4{0, 0, 0, 0};
    __syncthreads();
  }
  // this lane's places of a step: load i fills unit 64 (LPW wave + i) + lane
  auto place = [&](int i, int l, uint32_t& ko, uint32_t& vo, bool& kin, bool& vin) {
    const int pos = 64 * (LPW * wave + i) + l, row = pos / UNITS, u = pos % UNITS;
    const int ku = wide_k_unit<DP>(row, u), vu = wide_v_unit<DP>(row, u);
    kin = DP == D || 8 * ku < D;
    vin = DP == D || 8 * vu < D;
    ko = static_cast<uint32_t>(2 * (row * D + 8 * ku));
    vo = static_cast<uint32_t>(2 * (row * D + 8 * vu));
  };
  // (at head_dim over 128 no register is left to keep them: spilled, their reloads would wait for the loads in flight)
  constexpr bool kKeep = DP <= 128;
  uint32_t ko[kKeep ? LPW : 1], vo[kKeep ? LPW : 1];
  bool kin[kKeep ? LPW : 1], vin[kKeep ? LPW : 1];
  if constexpr (kKeep) {
#pragma unroll
    for (int i = 0; i < LPW; ++i) place(i, lane, ko[i], vo[i], kin[i], vin[i]);
  }
  // where this lane reads: K row n32 (+ 32), unit 2 ks + h; V row 4 h + (l16 >> 2) (+ 16 ks, + 8), channels
  // 32 cb + 16 ((lane >> 4) & 1) + 4 (l16 & 3), l16 = lane & 15.  Units are exchanged by an exclusive or within
  // 256 bytes, alike in rows 32, 16 and 8 apart: of an address, ks and cb change bits by one more of them, the
  // rest is a constant.
  constexpr int KA = NKS < 8 ? NKS : 8, VA = NCB < 4 ? NCB : 4;
  static_assert(TENSOR % 256 == 0, "rows start at multiples of the exchanged units' span");
  const int vrow = 4 * h + ((lane & 15) >> 2);
  uint32_t kat = base + n32 * DP * 2 + 16 * wide_k_unit<DP>(n32, h);
  uint32_t vat = base + TENSOR + vrow * DP * 2 + 16 * wide_v_unit<DP>(vrow, 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1)) + 8 * (lane & 1);
  int buf = 0;
  auto flip = [&]() {  // the next buffer
    const uint32_t d = buf == NST - 1 ? -static_cast<uint32_t>((NST - 1) * STAGE) : STAGE;
    kat += d;
    vat += d;
    buf = buf == NST - 1 ? 0 : buf + 1;
  };
  const float sl2 = p.scale_log2;
  // What a probability's exponent adds to the score's: the maximum's, and log2 of the factor on fp16 probabilities.
  // Far from zero both products are rounded by more than 1: the sum is kept from falling short (2^-22 of its size
  // covers three roundings), which would leave the maximum itself no weight, and where it exceeds by more than the
  // bound on probabilities, the scores' differences are taken first.
  constexpr float kHeld = BF ? 0.0f : 9.0f, kBound = BF ? 8.0f : 6.0f;
  auto held = [&](float m) {
    const float t = m * sl2;
    return fminf(fmaf(fabsf(t), 0x1p-22f, kHeld - t), 3.0e38f);
  };
  while (walk_next(p, KT, k)) {
    const Tile& w = k.w;
    const int all = w.n * p.G;  // the row's matrix rows
    auto limit = [&](int i) {
      const int x = p.causal ? w.len - w.n + i + 1 : w.len;
      return x < 0 ? 0 : x;
    };
    // this wave's matrix rows, and the fewest and the most keys they see
    const int r0 = w.tile * M + 32 * wave;
    const bool active = r0 < all;
    const int rl = r0 + 32 < all ? r0 + 32 : all;
    const int wlo = __builtin_amdgcn_readfirstlane(active ? limit(r0 / p.G) : 0);
    const int whi = __builtin_amdgcn_readfirstlane(active ? limit((rl - 1) / p.G) : 0);
    const const_i32* trow = (const const_i32*)(uintptr_t)(p.table + w.b * p.ppr);  // (scalar loads: vmcnt counts the steps' alone)
    auto issue = [&](int key, int id, int buf) {
      id = id < 0 || id >= p.n_pages ? 0 : id;
      const int64_t at = ((static_cast<int64_t>(id) * p.Hkv + kvh) * kPage + key % kPage) * D;
      const uint32_t to = base + buf * STAGE + 1024 * LPW * wave;
      if constexpr (kKeep) {
#pragma unroll
        for (int i = 0; i < LPW; ++i) {
          if (kin[i]) lds_dma16(p.kp + at, ko[i], to + 1024 * i);
          if (vin[i]) lds_dma16(p.vp + at, vo[i], to + TENSOR + 1024 * i);
        }
      } else {
        int l = threadIdx.x & 63;
        asm volatile("" : "+v"(l));  // (not computed ahead of the loop)
#pragma unroll
        for (int i = 0; i < LPW; ++i) {
          uint32_t k_off, v_off;
          bool k_in, v_in;
          place(i, l, k_off, v_off, k_in, v_in);
          if (k_in) lds_dma16(p.kp + at, k_off, to + 1024 * i);
          if (v_in) lds_dma16(p.vp + at, v_off, to + TENSOR + 1024 * i);
        }
      }
    };
    const bool live = r0 + n32 < all;
    // this lane's query and head (not kept over the steps, which need every register)
    auto row = [&](int& qi, int& hd) {
      int r = threadIdx.x & 31;
      asm volatile("" : "+v"(r));
      r = live ? r0 + r : 0;
      qi = r / p.G;
      hd = kvh * p.G + r - qi * p.G;
    };
    int lim;
    f32x16 acc[NCB];
    float m, l;  // of row n32: the running maximum (raw scores), the sum over this half's keys
    for (bool again = false;; again = true) {
      __syncthreads();  // the LDS is done with
      if (threadIdx.x == 0) any_nan = 0;
      int ahead = k.lo, next = 0;  // ahead: the first key not asked for
      auto issue_next = [&](int to) {
        issue(ahead, __builtin_amdgcn_readfirstlane(next), to);
        ahead += KT;
        if (ahead < k.hi) next = trow[ahead / kPage];
      };
      if (ahead < k.hi) {
        next = trow[ahead / kPage];
        issue_next(buf);
      }
      u32x4 qf[NKS];
      {
        int qi, hd;
        row(qi, hd);
        lim = live ? limit(qi) : 0;
        const uint16_t* qr = p.q + static_cast<int64_t>(w.q0 + qi) * p.q_st + static_cast<int64_t>(hd) * p.q_sh;
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) {
          const int c = 16 * ks + 8 * h;
          qf[ks] = live && c < D ? *reinterpret_cast<const u32x4*>(qr + c) : u32x4{0, 0, 0, 0};
        }
      }
      m = kNegBig;
      l = 0.0f;
#pragma unroll
      for (int cb = 0; cb < NCB; ++cb)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[cb][i] = 0.0f;

      // the query and the first step; in the loop only the direct loads are in flight, which the compiler does not count
      __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
#pragma unroll
      for (int i = 1; i < NST - 1; ++i)
        if (ahead < k.hi) issue_next(buf + i < NST ? buf + i : buf + i - NST);
      for (int key = k.lo; key < k.hi; key += KT, flip()) {
        // this wave's share of the step: later steps' may be in flight
        const int later = ahead - key - KT;
        if (NST > 3 && later > KT) __builtin_amdgcn_s_waitcnt(vmcnt_imm(4 * LPW));
        else if (NST > 2 && later > 0) __builtin_amdgcn_s_waitcnt(vmcnt_imm(2 * LPW));
        else __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
        __syncthreads();  // everyone's; and the step before is done with
        uint8_t* const vt = lds + buf * STAGE + TENSOR;
        const int cnt = w.len - key;
        if (cnt < KT) {  // rows that hold no token: whatever stands there must not count
          for (int i = threadIdx.x; i < (KT - cnt) * UNITS; i += 64 * NW) *reinterpret_cast<u32x4*>(vt + 16 * (cnt * UNITS + i)) = u32x4{0, 0, 0, 0};
          __syncthreads();
        }
        if (ahead < k.hi) issue_next(buf == 0 ? NST - 1 : buf - 1);
        const bool odd = again && Odd<BF>::template any<TENSOR / 1024>(vt, lane);
        if (key >= whi) {
          if (odd) {  // (the barriers of the waves that compute)
            __syncthreads();
            Odd<BF>::template clear<TENSOR, 64 * NW>(vt);
            __syncthreads();
          }
          continue;  // (to flip())
        }
        // fragments are read AH ahead of their products
        constexpr int AH = DP > 128 ? 2 : 4;
        constexpr int kCompute = 0x6;  // (vector and scalar arithmetic may pass, reads and products keep their order)
        auto k_frag = [&](int f) {  // k-step f / NKB of key block f % NKB
          const int ks = f / NKB;
          return lds_read16((kat ^ (32 * (ks % KA))) + 32 * (f % NKB) * DP * 2 + 256 * (ks / KA));
        };
        auto v_frag = [&](int f) {
          const uint32_t at = (vat ^ (64 * (f % NCB % VA))) + 16 * (f / NCB) * DP * 2 + 256 * (f % NCB / VA);
          const u32x2 w0 = lds_read_tr(at), w1 = lds_read_tr(at + 8 * DP * 2);  // (row + 8: the same exchange)
          return u32x4{w0.x, w0.y, w1.x, w1.y};
        };
        f32x16 s[NKB];
        {
          u32x4 kf[AH];
#pragma unroll
          for (int f = 0; f < AH; ++f) kf[f] = k_frag(f);
          __builtin_amdgcn_sched_barrier(kCompute);
#pragma unroll
          for (int f = 0; f < NKS * NKB; ++f) {
            const u32x4 a = kf[f % AH];
            if (f + AH < NKS * NKB) kf[f % AH] = k_frag(f + AH);
            if (f < NKB) {
#pragma unroll
              for (int i = 0; i < 16; ++i) s[f % NKB][i] = 0.0f;
            }
            s[f % NKB] = mfma32<BF>(a, qf[f / NKB], s[f % NKB]);
            __builtin_amdgcn_sched_barrier(kCompute);
          }
        }
        if (key + KT > wlo) {
          const int left = lim - key - 4 * h;
#pragma unroll
          for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (left <= 32 * kb + 8 * (i >> 2) + (i & 3)) s[kb][i] = -INFINITY;
        }
        u32x4 pa[2 * NKB];
        auto probs = [&](float nm) {
#pragma unroll
          for (int st = 0; st < 2 * NKB; ++st)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              pa[st][j] = pack2<BF>(__builtin_amdgcn_exp2f(fmaf(s[st >> 1][8 * (st & 1) + 2 * j], sl2, nm)),
                                    __builtin_amdgcn_exp2f(fmaf(s[st >> 1][8 * (st & 1) + 2 * j + 1], sl2, nm)));
        };
        probs(held(m));
        // 16-bit patterns of the non-negative probabilities order as their values do
        u16x8 pm = __builtin_elementwise_max(__builtin_bit_cast(u16x8, pa[0]), __builtin_bit_cast(u16x8, pa[1]));
        if constexpr (NKB == 2)
          pm = __builtin_elementwise_max(pm, __builtin_elementwise_max(__builtin_bit_cast(u16x8, pa[2]), __builtin_bit_cast(u16x8, pa[3])));
        const auto p2 = __builtin_elementwise_max(__builtin_elementwise_max(pm.s01, pm.s23), __builtin_elementwise_max(pm.s45, pm.s67));
        constexpr uint16_t kOver = BF ? 0x4380 : 0x7800;  // 2^8, 2^9 * 2^6
        const bool over = __builtin_amdgcn_ballot_w64(p2.x > kOver || p2.y > kOver) != 0;
        if (over || odd) {  // (one branch for what is rare)
          if (over) {
            float mx = kNegBig;
#pragma unroll
            for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
              for (int i = 0; i < 16; i += 2) mx = fmaxf(mx, fmaxf(s[kb][i], s[kb][i + 1]));
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
            const float mn = fmaxf(m, mx);
            float nm = held(mn);
            const float alpha = __builtin_amdgcn_exp2f(fminf(nm - held(m), 0.0f));
            m = mn;
            l *= alpha;
#pragma unroll
            for (int cb = 0; cb < NCB; ++cb)
#pragma unroll
              for (int i = 0; i < 16; ++i) acc[cb][i] *= alpha;
            const bool far = fmaf(m, sl2, nm) > kHeld + kBound + 0.25f;  // (0.25: a bound that rounding may have met is met here too)
            if (__builtin_amdgcn_ballot_w64(far) != 0) {
              const float less = far ? m : 0.0f;
              nm = far ? kHeld : nm;
#pragma unroll
              for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[kb][i] -= less;
            }
            probs(nm);
          }
          if (odd) {
#pragma unroll 1
            for (int j = 0; j < KT && key + j < lim; ++j)
#pragma unroll
              for (int cb = 0; cb < NCB; ++cb)
#pragma unroll
                for (int q = 0; q < 4; ++q) {  // channels 32 cb + 8 q + 4 h .. + 3
                  const u32x2 v = *reinterpret_cast<const u32x2*>(vt + j * DP * 2 + 16 * wide_v_unit<DP>(j, 4 * cb + q) + 8 * h);
#pragma unroll
                  for (int i = 0; i < 4; ++i) acc[cb][4 * q + i] = Odd<BF>::added(acc[cb][4 * q + i], v[i >> 1] >> (16 * (i & 1)));
                }
            __syncthreads();
            Odd<BF>::template clear<TENSOR, 64 * NW>(vt);
            __syncthreads();
          }
        }
        float ps = 0.0f;
#pragma unroll
        for (int st = 0; st < 2 * NKB; ++st)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t pw = pa[st][j];  // (a bit cast of a vector's element itself takes element 0)
            if constexpr (BF)
              ps = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pw), (bf16x2{static_cast<__bf16>(1.0f), static_cast<__bf16>(1.0f)}), ps, false);
            else
              ps = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, pw), (f16x2{static_cast<_Float16>(1.0f), static_cast<_Float16>(1.0f)}), ps, false);
          }
        l += ps;
        {
          u32x4 vf[AH];
#pragma unroll
          for (int f = 0; f < AH; ++f) vf[f] = v_frag(f);
          __builtin_amdgcn_sched_barrier(kCompute);
#pragma unroll
          for (int f = 0; f < 2 * NKB * NCB; ++f) {
            const u32x4 a = vf[f % AH];
            if (f + AH < 2 * NKB * NCB) vf[f % AH] = v_frag(f + AH);
            acc[f % NCB] = mfma32<BF>(a, pa[f / NCB], acc[f % NCB]);
            __builtin_amdgcn_sched_barrier(kCompute);
          }
        }
      }

      bool nan = false;
#pragma unroll
      for (int cb = 0; cb < NCB; ++cb)
#pragma unroll
        for (int i = 0; i < 16; ++i) nan |= acc[cb][i] != acc[cb][i];
      if (again) break;
      if (nan) any_nan = 1;
      __syncthreads();
      if (__builtin_amdgcn_readfirstlane(any_nan) == 0) break;
    }

    // ---- lane (n, h): row n, channels 32 cb + 8 q + 4 h .. + 3 ----
    const bool part = !(k.first && k.last);
    const float lt = l + __shfl_xor(l, 32, 64);
    if (live && part) {
      const int64_t pr = (static_cast<int64_t>(blockIdx.x) * 2 + (k.first ? 1 : 0)) * M + 32 * wave + n32;
      if (h == 0) p.part_ml[pr] = make_float2(-held(m), lt);
#pragma unroll
      for (int cb = 0; cb < NCB; ++cb)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int c = 32 * cb + 8 * q + 4 * h;
          if (c < D) *reinterpret_cast<f32x4*>(p.part_o + pr * D + c) = f32x4{acc[cb][4 * q], acc[cb][4 * q + 1], acc[cb][4 * q + 2], acc[cb][4 * q + 3]};
        }
    } else if (live) {
      const float inv = lt == 0.0f ? 0.0f : 1.0f / lt;  // no visible key: zeros
      int qi, hd;
      row(qi, hd);
      uint16_t* dst = p.out + static_cast<int64_t>(w.q0 + qi) * p.o_st + static_cast<int64_t>(hd) * p.o_sh;
#pragma unroll
      for (int cb = 0; cb < NCB; ++cb)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int c = 32 * cb + 8 * q + 4 * h;
          u32x2 o;
          o.x = pack2<BF>(acc[cb][4 * q] * inv, acc[cb][4 * q + 1] * inv);
          o.y = pack2<BF>(acc[cb][4 * q + 2] * inv, acc[cb][4 * q + 3] * inv);
          if (c < D) *reinterpret_cast<u32x2*>(dst + c) = o;
        }
    }
  }
  finish(p, k, true);
}

// Tiles that a piece's border cuts, their parts joined in the order of the keys:
// the beginning in piece `index` of the kv head, ends in the pieces after it.
// D / 4 threads per matrix row; of a tile of four parts or more four times as many,
// each with a share of the parts, whose sums are added up through LDS in a fixed order.
template <bool BF, int SHARES>
__device__ __forceinline__ void merge_rows(const Params& p, int block, const int4 cut, int row0, int row_step, f32x4* so, float2* sml) {
  const int parts = cut.w;
  const int kvh = block % p.Hkv, M = 1 << p.lm;
  const int rows = cut.z - cut.y < M ? cut.z - cut.y : M;
  const int tpr = p.D / 4, rows_at_once = kThreads / tpr / SHARES;
  const int grp = threadIdx.x / tpr, c = 4 * (threadIdx.x % tpr), sub = grp % SHARES;
  auto at = [&](int i, int row) { return ((static_cast<int64_t>(block) + static_cast<int64_t>(i) * p.Hkv) * 2 + (i == 0 ? 1 : 0)) * M + row; };
  for (int rb = row0 * rows_at_once; rb < rows; rb += row_step * rows_at_once) {
    const int row = rb + grp / SHARES;
    const bool mine = grp < rows_at_once * SHARES && row < rows;
    float mx = -INFINITY, sum = 0.0f;
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    if (mine) {
      // a running maximum, as in the kernels: the parts' loads do not wait for it
#pragma unroll 4
      for (int i = sub; i < parts; i += SHARES) {
        const float2 ml = p.part_ml[at(i, row)];
        const f32x4 a = *reinterpret_cast<const f32x4*>(p.part_o + at(i, row) * p.D + c);
        const float mn = fmaxf(mx, ml.x), ms = mn == -INFINITY ? 0.0f : mn;
        const float f0 = __builtin_amdgcn_exp2f(mx - ms), f1 = __builtin_amdgcn_exp2f(ml.x - ms);
        mx = mn;
        sum = sum * f0 + ml.y * f1;
        o = o * f0 + a * f1;
      }
    }
    if constexpr (SHARES > 1) {
      __syncthreads();
      so[threadIdx.x] = o;
      sml[threadIdx.x] = make_float2(mx, sum);
      __syncthreads();
      if (mine && sub == 0) {
        float2 ml[SHARES];
        f32x4 a[SHARES];
#pragma unroll
        for (int i = 0; i < SHARES; ++i) {
          ml[i] = sml[threadIdx.x + i * tpr];
          a[i] = so[threadIdx.x + i * tpr];
          mx = fmaxf(mx, ml[i].x);
        }
        const float ms = mx == -INFINITY ? 0.0f : mx;
        sum = 0.0f;
        o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < SHARES; ++i) {
          const float f = __builtin_amdgcn_exp2f(ml[i].x - ms);
          sum += ml[i].y * f;
          o += a[i] * f;
        }
      }
    }
    if (mine && sub == 0) {
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      const int r = cut.y + row, qi = r / p.G;
      uint16_t* dst = p.out + static_cast<int64_t>(cut.x + qi) * p.o_st + static_cast<int64_t>(kvh * p.G + r - qi * p.G) * p.o_sh + c;
      *reinterpret_cast<u32x2*>(dst) = u32x2{pack2<BF>(o[0] * inv, o[1] * inv), pack2<BF>(o[2] * inv, o[3] * inv)};
    }
  }
}
template <bool BF>
__device__ __forceinline__ void merge_tile(const Params& p, int block, int row0, int row_step) {
  const int4 cut = p.cuts[block];
  if (cut.w < 2) return;
  __shared__ f32x4 so[kThreads];
  __shared__ float2 sml[kThreads];
  if (cut.w < 4) merge_rows<BF, 1>(p, block, cut, row0, row_step, so, sml);
  else merge_rows<BF, 4>(p, block, cut, row0, row_step, so, sml);  // (D / 4 threads four times fit a block)
}

// Sixteen blocks per piece of the wide kernel, whose tiles take longer to join, then four per piece of the few-row
// kernel (8 and 8, the few-row kernel's first: 30 decoding rows with two 512-token chunks 222 us, now 218; decoding
// rows alone 155.4 and 153.1).
constexpr int kWideBlocks = 16, kFewBlocks = 4;
template <bool BF>
__global__ __launch_bounds__(kThreads) void paged_merge_kernel(Params wide, Params few, int wide_blocks) {
  const int i = blockIdx.x, j = i - wide_blocks;
  if (j < 0) merge_tile<BF>(wide, i / kWideBlocks, i % kWideBlocks, kWideBlocks);
  else merge_tile<BF>(few, j / kFewBlocks, j % kFewBlocks, kFewBlocks);
}

bool aligned16(const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15) == 0; }

template <int DP>
struct Wide {  // waves, matrix rows, keys per step, steps' buffers
  static constexpr int NW = 8, M = 32 * NW, KT = DP > 128 ? 32 : 64, NST = DP > 128 ? 4 : 3;
};
constexpr int kWideLog = 8;

// The two kernels' cuts of a call.
struct Plan {
  Params few, wide;
  bool both;  // the wide kernel runs too
};

void set_cut(Params& p, int rows_of, int lm, int start_cost, int64_t workgroups, int least, int snap) {
  p.rows_of = rows_of;
  p.lm = lm;
  p.per_tile = static_cast<int>(cdiv(1 << lm, p.G));
  p.start_cost = start_cost;
  p.least = least;
  p.snap = snap;
  // pieces: no more than the longest line that the tensors allow has of the least size
  const int64_t tiles = p.T * p.G / (1 << lm) + (p.B < p.T ? p.B : p.T);
  const int64_t line = tiles * (p.ppr * kPage + p.start_cost + p.per_tile);
  int64_t n = workgroups / p.Hkv;
  if (n > cdiv(line, least)) n = cdiv(line, least);
  p.pieces = static_cast<int>(n < 1 ? 1 : n);
  p.per_piece = 1.00002f / static_cast<float>(p.pieces);
}

int plan_of(const fade_paged_attn_args* a, Plan& pl) {
  const char* what = "fade_paged_attn";
  if (a == nullptr) return einval("%s: null args", what);
  if (a->D < 8 || a->D > 256 || a->D % 8)
    return einval("%s: head_dim must be a multiple of 8 in [8, 256], got %lld", what, (long long)a->D);
  if (a->B < 1 || a->T < 0 || a->Hq < 1 || a->Hkv < 1 || a->n_pages < 1 || a->pages_per_row < 1)
    return einval("%s: B, Hq, Hkv, n_pages and pages_per_row must be positive, T not negative", what);
  if (a->Hq % a->Hkv) return einval("%s: needs Hq %% Hkv == 0 (got %lld/%lld)", what, (long long)a->Hq, (long long)a->Hkv);
  if (a->B > (1 << 20) || a->T > (1 << 24) || a->Hq > 65535 || a->T * (a->Hq / a->Hkv) >= (1ll << 30) ||
      a->pages_per_row > (1 << 24) || a->n_pages >= (1ll << 31))
    return einval("%s: shape too large", what);
  if (a->T > 0 && (!a->q || !a->out)) return einval("%s: null q or out", what);
  if (!a->k_pages || !a->v_pages || !a->table || !a->lens || !a->starts) return einval("%s: null pages, table, lens or starts", what);
  if (!aligned16(a->q) || (a->q_st | a->q_sh) % 8) return einval("%s: q rows must be 16-byte aligned", what);
  if ((reinterpret_cast<uintptr_t>(a->out) & 7) || (a->o_st | a->o_sh) % 4) return einval("%s: out rows must be 8-byte aligned", what);
  if (!aligned16(a->k_pages) || !aligned16(a->v_pages)) return einval("%s: pages must be 16-byte aligned", what);
  if (a->dtype != FADE_DTYPE_F16 && a->dtype != FADE_DTYPE_BF16)
    return einval("%s: dtype must be FADE_DTYPE_F16 or FADE_DTYPE_BF16, got %d", what, a->dtype);
  if (a->mask_mode != FADE_MASK_BOTTOM_RIGHT && a->mask_mode != FADE_MASK_NONE)
    return einval("%s: mask_mode must be FADE_MASK_BOTTOM_RIGHT or FADE_MASK_NONE, got %d", what, a->mask_mode);
  if (!(a->sm_scale > 0.0f) || !(a->sm_scale < INFINITY)) return einval("%s: sm_scale must be positive and finite", what);
  Params p{};
  p.B = a->B;
  p.T = a->T;
  p.ppr = a->pages_per_row;
  p.n_pages = a->n_pages;
  p.Hq = static_cast<int>(a->Hq);
  p.Hkv = static_cast<int>(a->Hkv);
  p.G = p.Hq / p.Hkv;
  p.D = static_cast<int>(a->D);
  p.q = static_cast<const uint16_t*>(a->q);
  p.q_st = a->q_st;
  p.q_sh = a->q_sh;
  p.out = static_cast<uint16_t*>(a->out);
  p.o_st = a->o_st;
  p.o_sh = a->o_sh;
  p.kp = static_cast<const uint16_t*>(a->k_pages);
  p.vp = static_cast<const uint16_t*>(a->v_pages);
  p.table = a->table;
  p.lens = a->lens;
  p.starts = a->starts;
  p.scale_log2 = a->sm_scale * 1.4426950408889634f;
  p.causal = a->mask_mode == FADE_MASK_BOTTOM_RIGHT;
  p.zero_tail = a->zero_tail;
  // Rows whose matrix rows fit one tile of 16 go to the few-row kernel, the others
  // to the wide one (16 rows over 8192 keys each, 32 matrix rows a row: 113 us, by the
  // few-row kernel 124; 64: 114 and 204; 128: 131 and 389).  The host does not know the
  // rows, and the wide kernel's launch, empty, costs a decoding step 2 to 5 us (64 rows of
  // 1000 keys 54 us, with it 59; one row of 1000 keys 10.9 and 13.0), so a step goes to the
  // few-row kernel as a whole where no row of it can be longer while the others have a
  // token each.  A chunk taken for a part of such a step costs far more: 63 rows of 1000
  // keys beside 193 tokens over 8192 keys 201 us, 117 by both kernels; 900 tokens at 32 kv
  // heads 895 and 352.  Rows without tokens can still hide one (64 of them, 64 tokens over
  // 8192 keys 67 us and 45, over 1000 keys 27 and 36), so it is bound to four wide tiles.
  const bool step = (p.T - p.B + 1) * p.G <= kRows && p.T * p.G <= 1024;
  pl.both = !step;
  // The few-row kernel has as many workgroups as find a place at once (16 rows over
  // 8192 keys: 4 per CU 104.5 us, 8 110.6, 16 120), of 64 keys or more each (a row of
  // 1000 keys: 32 and 64 alike, 128 2 us more, 256 4); the wide one a workgroup per CU (30 decoding
  // rows with two 512-token chunks: 241 us, two 280, three 291), a tile's start and end
  // counted as 300 keys (a prompt of 4096 tokens 184 us, four of 1000 at head_dim 256
  // 84; as 192: 200 and 97, as 500: 182 and 96, and eight of 512 74 instead of 61), and a
  // border within 256 keys of a tile's, and a third of a piece, moved there: the fp32
  // sums of a cut tile cost as much (three prompts at head_dim 256 134 us, unmoved 151;
  // eight of 512 tokens 61 and 77; long chunks alike).
  const int per_cu = p.D <= 64 ? 8 : (p.D <= 128 ? 4 : 2);
  pl.few = pl.wide = p;
  set_cut(pl.few, step ? kAll : kFew, 4, 32, static_cast<int64_t>(per_cu) * num_cus(), 64, 0);
  set_cut(pl.wide, kMany, kWideLog, 300, num_cus(), 256, 256);
  pl.wide.zero_tail = 0;
  return FADE_OK;
}

int64_t part_rows(const Params& p) { return p.pieces < 2 ? 0 : static_cast<int64_t>(p.pieces) * p.Hkv * 2 << p.lm; }
int64_t part_rows(const Plan& pl) { return part_rows(pl.few) + (pl.both ? part_rows(pl.wide) : 0); }
int64_t cut_bytes(const Params& p) { return static_cast<int64_t>(p.pieces) * p.Hkv * static_cast<int64_t>(sizeof(int4)); }
int64_t part_bytes(const Plan& pl) {
  const int64_t n = part_rows(pl);
  return n == 0 ? 0 : cut_bytes(pl.few) + cut_bytes(pl.wide) + n * (pl.few.D * 4 + static_cast<int64_t>(sizeof(float2)));
}

template <int DP, bool BF>
int launch(const Plan& pl, hipStream_t st) {
  if (pl.both) {
    typedef Wide<DP> W;
    hipLaunchKernelGGL((paged_wide_kernel<DP, W::NW, W::KT, W::NST, BF>), dim3(static_cast<unsigned>(pl.wide.Hkv * pl.wide.pieces)), dim3(64 * W::NW), 0, st, pl.wide);
    const int rc = check_launch("fade_paged_attn");
    if (rc) return rc;
  }
  hipLaunchKernelGGL((paged_few_kernel<DP, BF>), dim3(static_cast<unsigned>(pl.few.Hkv * pl.few.pieces)), dim3(64), 0, st, pl.few);
  const int rc = check_launch("fade_paged_attn");
  // (the last piece's tiles end in it)
  const int wide = pl.both ? pl.wide.Hkv * (pl.wide.pieces - 1) * kWideBlocks : 0, few = pl.few.Hkv * (pl.few.pieces - 1) * kFewBlocks;
  if (rc || wide + few == 0) return rc;
  hipLaunchKernelGGL((paged_merge_kernel<BF>), dim3(static_cast<unsigned>(wide + few)), dim3(kThreads), 0, st, pl.wide, pl.few, wide);
  return check_launch("fade_paged_attn (merge)");
}

template <bool BF>
int launch_any(const Plan& pl, void* stream) {
  hipStream_t st = as_stream(stream);
  if (pl.few.D <= 64) return launch<64, BF>(pl, st);
  if (pl.few.D <= 128) return launch<128, BF>(pl, st);
  return launch<256, BF>(pl, st);
}

}  // namespace
}  // namespace paged
}  // namespace fade

using namespace fade;
using namespace fade::paged;

FADE_API int fade_paged_attn_workspace_bytes(const fade_paged_attn_args* a, int64_t* bytes) {
  if (bytes == nullptr) return einval("fade_paged_attn_workspace_bytes: null output");
  Plan pl;
  const int rc = plan_of(a, pl);
  if (rc) return rc;
  *bytes = part_bytes(pl);
  return FADE_OK;
}

FADE_API int fade_paged_attn(const fade_paged_attn_args* a, void* workspace, int64_t workspace_bytes, void* stream) {
  Plan pl;
  const int rc = plan_of(a, pl);
  if (rc) return rc;
  if (a->T == 0) return FADE_OK;
  const int64_t need = part_bytes(pl);
  if (need > 0) {
    if (workspace == nullptr || workspace_bytes < need || !aligned16(workspace))
      return einval("fade_paged_attn: needs a 16-byte aligned workspace of %lld bytes", (long long)need);
    const int64_t all = part_rows(pl), few = part_rows(pl.few);
    pl.few.cuts = static_cast<int4*>(workspace);
    pl.wide.cuts = pl.few.cuts + cut_bytes(pl.few) / sizeof(int4);
    pl.few.part_o = reinterpret_cast<float*>(pl.wide.cuts + cut_bytes(pl.wide) / sizeof(int4));
    pl.few.part_ml = reinterpret_cast<float2*>(pl.few.part_o + all * pl.few.D);
    pl.wide.part_o = pl.few.part_o + few * pl.few.D;
    pl.wide.part_ml = pl.few.part_ml + few;
  }
  return a->dtype == FADE_DTYPE_BF16 ? launch_any<true>(pl, stream) : launch_any<false>(pl, stream);
}
