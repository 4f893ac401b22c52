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
// Work is cut on the device, from the lengths the host does not know: an item is
// (row b, tile of M matrix rows, split of the keys), and a split holds
// C = max(kLeast, ceil(sum_b tiles_b L_b / target)) keys, so that the items are about
// `target` equal pieces whatever the rows' lengths are.  Every wave finds its own
// item by a sum over the rows' counts (one load per lane for 64 rows).  A row that
// is one split writes its output; the others' unnormalized fp32 sums are joined in
// split order by a second launch, so results do not depend on timing.
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
constexpr float kNegBig = -1.0e30f;

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
  int target;      // items per kv head the splits aim at; 0: no splits
  float per_item;  // a little over 1 / target
  uint32_t items;  // bound of the items per kv head
  int rows_of;     // kAll, or the rows of the batch whose matrix rows fit one tile of 16 (kFew) or do not (kMany)
  int least;       // fewest keys of a split (a multiple of 64)
  float* part_o;   // [item][kv head][M][D]
  float2* part_ml; // [item][kv head][M]: maximum (log2 units), sum
};

// What a wave works on (wave-uniform).
struct Item {
  int b, q0, n, len;    // row, its first new token, new tokens, tokens
  int tile, split;      // tile of matrix rows, split of the keys
  int tiles, splits;    // the row's
  int chunk;            // keys per split
  uint32_t first;       // the row's first item
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

// Inclusive sums over the wave's lanes: shifts within rows of 16 lanes, then each
// row's last lane to the next row (DPP: no LDS round trips).
template <typename T, typename F>
__device__ __forceinline__ T wave_scan(T v, F add) {
  auto step = [&](auto ctrl, auto mask) {
    const int x = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), decltype(ctrl)::value, decltype(mask)::value, 0xF, true);
    v = add(v, __builtin_bit_cast(T, x));
  };
  step(Int<0x111>{}, Int<0xF>{});  // row_shr 1, 2, 4, 8
  step(Int<0x112>{}, Int<0xF>{});
  step(Int<0x114>{}, Int<0xF>{});
  step(Int<0x118>{}, Int<0xF>{});
  step(Int<0x142>{}, Int<0xA>{});  // row_bcast 15 to rows 1 and 3
  step(Int<0x143>{}, Int<0xC>{});  // row_bcast 31 to rows 2 and 3
  return v;
}
__device__ __forceinline__ uint32_t scan_u32(uint32_t v) {
  return wave_scan(v, [](uint32_t a, uint32_t b) { return a + b; });
}
__device__ __forceinline__ float sum_f32(float v) {
  const float x = wave_scan(v, [](float a, float b) { return __fadd_rn(a, b); });
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 63));
}
__device__ __forceinline__ uint32_t lane_of(uint32_t v, int l) {
  return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), l));
}

// Item `idx` (BY_TILE: the idx-th tile of rows, all its splits) of a kernel of M
// matrix rows; false past the last one.  All lanes of the wave call it.
template <int M, bool BY_TILE>
__device__ __forceinline__ bool find_item(const Params& p, uint32_t idx, Item& it) {
  const int lane = threadIdx.x & 63;
  const int B = static_cast<int>(p.B);
  int q0 = 0, n = 0, len = 0;
  auto tiles_of = [&](int new_tokens) {
    const uint32_t rows = static_cast<uint32_t>(new_tokens) * static_cast<uint32_t>(p.G);
    if (p.rows_of != kAll && (rows <= kRows) != (p.rows_of == kFew)) return 0u;
    return (rows + static_cast<uint32_t>(M - 1)) / static_cast<uint32_t>(M);
  };
  uint32_t chunk = INT32_MAX;
  if (p.target > 0) {
    // (every wave of both launches does the same operations in the same order; the
    // factor keeps chunk * target at or above the work despite the roundings)
    float work = 0.0f;
    for (int b = lane; b < B; b += 64) {
      row_counts(p, b, q0, n, len);
      work = __fmaf_rn(static_cast<float>(tiles_of(n)), static_cast<float>(len), work);
    }
    work = __fmul_rn(sum_f32(work), p.per_item);
    const uint32_t c = work < 1.0e9f ? static_cast<uint32_t>(work) + 1u : 1000000000u;
    chunk = (c + (kPage - 1)) / kPage * kPage;
    if (chunk < static_cast<uint32_t>(p.least)) chunk = static_cast<uint32_t>(p.least);
    chunk = __builtin_amdgcn_readfirstlane(chunk);
  }
  uint32_t items = 0, tiles_before = 0;
  for (int b0 = 0; b0 < B; b0 += 64) {
    const int b = b0 + lane;
    uint32_t tiles = 0, splits = 1;
    if (b < B) {
      if (B > 64 || p.target == 0) row_counts(p, b, q0, n, len);
      tiles = tiles_of(n);
      if (static_cast<uint32_t>(len) > chunk) splits = (static_cast<uint32_t>(len) + chunk - 1) / chunk;
    }
    const uint32_t cnt = tiles * splits;
    const uint32_t to_items = items + scan_u32(cnt), to_tiles = tiles_before + scan_u32(tiles);
    const bool mine = BY_TILE ? (idx < to_tiles && idx >= to_tiles - tiles) : (idx < to_items && idx >= to_items - cnt);
    const uint64_t who = __builtin_amdgcn_ballot_w64(mine);
    if (who != 0) {
      const int l = __builtin_ctzll(who);
      it.b = b0 + l;
      it.q0 = __builtin_amdgcn_readlane(q0, l);
      it.n = __builtin_amdgcn_readlane(n, l);
      it.len = __builtin_amdgcn_readlane(len, l);
      it.tiles = static_cast<int>(lane_of(tiles, l));
      it.splits = static_cast<int>(lane_of(splits, l));
      it.first = lane_of(to_items - cnt, l);
      it.chunk = static_cast<int>(chunk);
      const uint32_t rem = idx - (BY_TILE ? lane_of(to_tiles - tiles, l) : it.first);
      const uint32_t t = BY_TILE ? rem : rem / static_cast<uint32_t>(it.splits);
      it.tile = it.tiles - 1 - static_cast<int>(t);  // the last rows first: they see the most keys
      it.split = BY_TILE ? 0 : static_cast<int>(rem - t * static_cast<uint32_t>(it.splits));
      return true;
    }
    items = lane_of(to_items, 63);
    tiles_before = lane_of(to_tiles, 63);
  }
  return false;
}

// Rows of q past the last sequence: zeros, where the caller asked for them.
__device__ __forceinline__ void zero_tail(const Params& p, int64_t block, int64_t blocks, int kvh) {
  int end = p.starts[p.B];
  end = end < 0 ? 0 : end;
  const int G = p.G;
  for (int64_t t = end + block; t < p.T; t += blocks)
    for (int i = threadIdx.x; i < G * p.D; i += blockDim.x)
      p.out[t * p.o_st + (static_cast<int64_t>(kvh) * G + i / p.D) * p.o_sh + i % p.D] = 0;
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

// ---- few rows: tiles of 16 matrix rows, every wave with keys of its own ----
//
// A wave takes every fourth (head_dim over 128: second) tile of 32 keys of the
// item's split.  K and V rows go
// from the page straight to the wave's own LDS (no register holds them, no barrier
// is needed), two tiles deep: the next tile's loads fly while this one is computed.
//   S^T = K Q^T   16x16x32 MFMAs, A = 16 keys x 32 channels, B = Q^T (registers):
//                 lane (n, g) holds query row n, keys 4 g + i of the 16
//   O^T += V^T P^T  A = V^T by transposing LDS reads (4 keys x 16 channels each),
//                 B = P^T straight from S^T's registers: k slot (g, j) is key
//                 4 g + j of the first 16 keys (j < 4), 4 g + j - 4 of the second
// so the running maximum, the sum and the rescaling are lane-local; P is multiplied
// as a 16-bit head plus a 16-bit rest (P to 2^-16 or better): the matrix cores are
// idle here, and rounding P alone would cost as much accuracy as rounding the output.
// 16-byte unit u of LDS row r lies at unit u ^ (2 (r & 7)) (mod the row), which the
// loads' source addresses bring about: without it the 16 rows that a transposing
// read touches would share their banks.
template <int DP>
struct Few {
  static constexpr int kKeys = 32;                 // keys per tile
  static constexpr int kUnits = DP / 8;            // 16-byte units per row
  static constexpr int kTensor = kKeys * DP * 2;   // bytes of a tile's K or V
  static constexpr int kStage = 2 * kTensor;
  static constexpr int kLoads = kStage / 1024;     // direct loads per tile
  static constexpr int kWaves = DP > 128 ? 2 : 4;  // (a workgroup's LDS)
  static constexpr int kLds = kWaves * 2 * kStage;
  static constexpr int kSwizzle = kUnits - 1;
};

template <int DP>
__device__ __forceinline__ int few_unit(int row, int u) {
  return u ^ ((2 * row) & Few<DP>::kSwizzle);
}

template <int DP, bool BF>
__global__ __launch_bounds__(64 * Few<DP>::kWaves) void paged_few_kernel(Params p) {
  typedef Few<DP> F;
  constexpr int NKS = DP / 32, NCB = DP / 16, NW = F::kWaves;
  const int kvh = blockIdx.x % p.Hkv;
  const uint32_t idx = blockIdx.x / static_cast<uint32_t>(p.Hkv);
  const int lane = threadIdx.x & 63, n16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (p.zero_tail) zero_tail(p, idx, gridDim.x / p.Hkv, kvh);
  Item it;
  if (!find_item<kRows, false>(p, idx, it)) return;
  const int D = p.D;
  const int rows = it.n * p.G - it.tile * kRows < kRows ? it.n * p.G - it.tile * kRows : kRows;
  // this lane's matrix row: its query, head and visible keys
  const int r = it.tile * kRows + n16;
  const bool live = n16 < rows;
  const int qi = live ? r / p.G : 0, hd = kvh * p.G + (live ? r - qi * p.G : 0);
  auto limit = [&](int i) {
    const int x = p.causal ? it.len - it.n + i + 1 : it.len;
    return x < 0 ? 0 : x;
  };
  const int lim = live ? limit(qi) : 0;
  const int lo = limit(it.tile * kRows / p.G), hi = limit((it.tile * kRows + rows - 1) / p.G);  // fewest, most keys of the tile's rows
  const int k0 = __builtin_amdgcn_readfirstlane(it.split * it.chunk);  // (chunk INT32_MAX: split 0)
  const int k1 = __builtin_amdgcn_readfirstlane(it.splits > 1 && k0 + it.chunk < hi ? k0 + it.chunk : hi);

  __shared__ __attribute__((aligned(16))) uint8_t lds[F::kLds];
  uint8_t* const mine = &lds[wave * 2 * F::kStage];
  const uint32_t base = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_u8*)mine)));
  if (D < DP) {  // units past the head_dim are never loaded: zeros
    for (int i = 16 * lane; i < 2 * F::kStage; i += 1024) *reinterpret_cast<u32x4*>(mine + i) = u32x4{0, 0, 0, 0};
    __builtin_amdgcn_s_waitcnt(kLgkm0);
  }

  f32x4 acc[NCB];
#pragma unroll
  for (int cb = 0; cb < NCB; ++cb) acc[cb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float m = -INFINITY, l = 0.0f;  // of row n16 (l: over this lane's keys)

  const const_i32* trow = (const const_i32*)(uintptr_t)(p.table + it.b * p.ppr);  // (scalar loads: vmcnt counts the tiles' alone)
  auto page_at = [&](int key) {
    const int id = __builtin_amdgcn_readfirstlane(trow[key / kPage]);
    return static_cast<int64_t>(id < 0 || id >= p.n_pages ? 0 : id);
  };
  auto issue = [&](int key, int64_t page, int buf) {
    const int64_t at = ((page * p.Hkv + kvh) * kPage + key % kPage) * D;
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
  const int step = NW * F::kKeys;
  int key = k0 + wave * F::kKeys;
  int64_t next_page = 0;
  if (key < k1) {
    issue(key, page_at(key), 0);
    if (key + step < k1) next_page = page_at(key + step);
  }
  u32x4 qf[NKS];
  const uint16_t* qr = p.q + static_cast<int64_t>(it.q0 + qi) * p.q_st + static_cast<int64_t>(hd) * p.q_sh;
#pragma unroll
  for (int ks = 0; ks < NKS; ++ks) {
    const int c = 32 * ks + 8 * g;
    qf[ks] = live && c < D ? *reinterpret_cast<const u32x4*>(qr + c) : u32x4{0, 0, 0, 0};
  }
  // the query and the first tile; in the loop only the direct loads are in flight, which the compiler does not count
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
  for (int t = 0; key < k1; key += step, t ^= 1) {
    if (key + step < k1) {
      issue(key + step, next_page, t ^ 1);
      __builtin_amdgcn_s_waitcnt(vmcnt_imm(F::kLoads));
      if (key + 2 * step < k1) next_page = page_at(key + 2 * step);
    } else {
      __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
    }
    asm volatile("" ::: "memory");
    uint8_t* const kt = mine + t * F::kStage;
    uint8_t* const vt = kt + F::kTensor;
    const int cnt = it.len - key;  // rows from here on hold no token of the row: whatever stands there must not count
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
    const bool whole = key + F::kKeys <= lo;
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
    const float alpha = __builtin_amdgcn_exp2f(m - ms);
    m = mn;
    float ps = 0.0f;
    u32x4 ph, pl;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const float a = __builtin_amdgcn_exp2f(x[i] - ms), b = __builtin_amdgcn_exp2f(x[i + 1] - ms);
      ps += a + b;
      const uint32_t h = pack2<BF>(a, b);
      ph[i / 2] = h;
      pl[i / 2] = pack2<BF>(a - w2f<BF>(static_cast<uint16_t>(h)), b - w2f<BF>(static_cast<uint16_t>(h >> 16)));
    }
    l = l * alpha + ps;
#pragma unroll
    for (int cb = 0; cb < NCB; ++cb) {
      // lane (n, g) points at key 4 g + n / 4 (+ 16), channels 16 cb + 4 (n % 4) .. + 3
      const int row = 4 * g + (n16 >> 2), u = 2 * cb + ((n16 >> 1) & 1);
      const uint8_t* at = vt + row * DP * 2 + 16 * few_unit<DP>(row, u) + 8 * (n16 & 1);
      const i16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_i16x4*>((lds_u8*)const_cast<uint8_t*>(at)));
      const i16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          reinterpret_cast<lds_i16x4*>((lds_u8*)const_cast<uint8_t*>(at + 16 * DP * 2)));  // (row + 16: the same swizzle)
      const u32x2 w0 = __builtin_bit_cast(u32x2, v0), w1 = __builtin_bit_cast(u32x2, v1);
      const u32x4 a = {w0.x, w0.y, w1.x, w1.y};
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[cb][i] *= alpha;
      acc[cb] = mfma16<BF>(a, ph, acc[cb]);
      acc[cb] = mfma16<BF>(a, pl, acc[cb]);
    }
  }
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);

  // ---- the waves' sums joined, in wave order ----
  constexpr int PITCH = DP + 4;
  static_assert(NW * kRows * PITCH * 4 <= F::kLds, "the waves' sums fit the tiles' LDS");
  float* const so = reinterpret_cast<float*>(lds);
  __shared__ float2 sml[NW][kRows];
  __syncthreads();
#pragma unroll
  for (int cb = 0; cb < NCB; ++cb) *reinterpret_cast<f32x4*>(so + (wave * kRows + n16) * PITCH + 16 * cb + 4 * g) = acc[cb];
  if (g == 0) sml[wave][n16] = make_float2(m, l);
  __syncthreads();
  const bool part = it.splits > 1;
  const int64_t pr = static_cast<int64_t>(blockIdx.x) * kRows;
  for (int i = threadIdx.x; i < rows * (DP / 4); i += 64 * NW) {
    const int row = i / (DP / 4), c = 4 * (i % (DP / 4));
    if (c >= D) continue;
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) mx = fmaxf(mx, sml[w][row].x);
    const float ms = mx == -INFINITY ? 0.0f : mx;
    float sum = 0.0f;
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float f = __builtin_amdgcn_exp2f(sml[w][row].x - ms);
      sum += sml[w][row].y * f;
      o += *reinterpret_cast<const f32x4*>(so + (w * kRows + row) * PITCH + c) * f;
    }
    if (part) {
      *reinterpret_cast<f32x4*>(p.part_o + (pr + row) * D + c) = o;
      if (c == 0) p.part_ml[pr + row] = make_float2(mx, sum);
    } else {
      const int rr = it.tile * kRows + row, qq = rr / p.G;
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;  // no visible key: zeros
      uint16_t* dst = p.out + static_cast<int64_t>(it.q0 + qq) * p.o_st + static_cast<int64_t>(kvh * p.G + rr - qq * p.G) * p.o_sh + c;
      u32x2 w;
      w.x = static_cast<uint32_t>(f2w<BF>(o[0] * inv)) | (static_cast<uint32_t>(f2w<BF>(o[1] * inv)) << 16);
      w.y = static_cast<uint32_t>(f2w<BF>(o[2] * inv)) | (static_cast<uint32_t>(f2w<BF>(o[3] * inv)) << 16);
      *reinterpret_cast<u32x2*>(dst) = w;
    }
  }
}

// ---- many rows: tiles of 32 NW MT matrix rows, the keys shared through LDS ----
//
// NW waves of MT blocks of 32 matrix rows each walk the item's keys page by page.
// A page's K and V go straight to LDS, two pages deep, every wave loading its
// share; one barrier per page.
//   S^T = K Q^T   32x32x16 MFMAs, A = 32 keys x 16 channels, B = Q^T (registers):
//                 lane (n, h) holds matrix row n, register i key 8 (i / 4) + 4 h + i % 4
//   O^T += V^T P^T  A = V^T by transposing LDS reads, B = P^T straight from S^T's
//                 registers: k slot (h, j) of step s is key 16 s + 4 h + j (j < 4),
//                 16 s + 8 + 4 h + j - 4
// so a row's maximum, sum and rescaling are lane-local.  The running maximum moves
// only where a probability passes 2^8 (found on the 16-bit probabilities, two per
// operation; the exact maximum is taken there alone), so most pages need neither a
// maximum of the scores nor an exchange between lanes nor a rescaling.  P is
// rounded to 16 bits (as the output is; the sum takes the same rounded values): a
// second product for its rest would cost half the matrix work again.
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
template <bool BF>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <int DP, int NW, int MT, bool BF>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(NW / 4, NW / 4))) void paged_wide_kernel(Params p) {
  constexpr int M = 32 * NW * MT;
  constexpr int NKS = DP / 16, NCB = DP / 32, UNITS = DP / 8;
  constexpr int TENSOR = kPage * DP * 2, STAGE = 2 * TENSOR;
  constexpr int LPW = TENSOR / 1024 / NW;  // direct loads of K, and of V, per wave and page
  static_assert(TENSOR % (1024 * NW) == 0, "a page is shared out evenly");
  const int kvh = blockIdx.x % p.Hkv;
  const uint32_t idx = blockIdx.x / static_cast<uint32_t>(p.Hkv);
  const int lane = threadIdx.x & 63, n32 = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (p.zero_tail) zero_tail(p, idx, gridDim.x / p.Hkv, kvh);
  Item it;
  if (!find_item<M, false>(p, idx, it)) return;
  const int D = p.D;
  const int all = it.n * p.G;  // the row's matrix rows
  auto limit = [&](int i) {
    const int x = p.causal ? it.len - it.n + i + 1 : it.len;
    return x < 0 ? 0 : x;
  };
  const int last = it.tile * M + M < all ? it.tile * M + M : all;  // past the item's last matrix row
  const int hi = limit((last - 1) / p.G);
  const int k0 = __builtin_amdgcn_readfirstlane(it.split * it.chunk);
  const int k1 = __builtin_amdgcn_readfirstlane(it.splits > 1 && k0 + it.chunk < hi ? k0 + it.chunk : hi);
  // this wave's matrix rows, and the fewest and the most keys they see
  const int r0 = it.tile * M + 32 * MT * wave;
  const bool active = r0 < all;
  const int rl = r0 + 32 * MT < all ? r0 + 32 * MT : all;
  const int wlo = __builtin_amdgcn_readfirstlane(active ? limit(r0 / p.G) : 0);
  const int whi = __builtin_amdgcn_readfirstlane(active ? limit((rl - 1) / p.G) : 0);
  int lim[MT];

  __shared__ __attribute__((aligned(16))) uint8_t lds[2 * STAGE];
  const uint32_t base = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_u8*)lds)));
  if (D < DP) {  // units past the head_dim are never loaded: zeros
    for (int i = 16 * threadIdx.x; i < 2 * STAGE; i += 1024 * NW) *reinterpret_cast<u32x4*>(lds + i) = u32x4{0, 0, 0, 0};
    __syncthreads();
  }
  // this lane's places of a page: load i fills unit 64 (LPW wave + i) + lane
  uint32_t ko[LPW], vo[LPW];
  bool kin[LPW], vin[LPW];
#pragma unroll
  for (int i = 0; i < LPW; ++i) {
    const int pos = 64 * (LPW * wave + i) + lane, row = pos / UNITS, u = pos % UNITS;
    const int ku = wide_k_unit<DP>(row, u), vu = wide_v_unit<DP>(row, u);
    kin[i] = DP == D || 8 * ku < D;
    vin[i] = DP == D || 8 * vu < D;
    ko[i] = static_cast<uint32_t>(2 * (row * D + 8 * ku));
    vo[i] = static_cast<uint32_t>(2 * (row * D + 8 * vu));
  }
  const const_i32* trow = (const const_i32*)(uintptr_t)(p.table + it.b * p.ppr);
  auto issue = [&](int id, int buf) {
    id = id < 0 || id >= p.n_pages ? 0 : id;
    const int64_t at = (static_cast<int64_t>(id) * p.Hkv + kvh) * kPage * D;
    const uint32_t to = base + buf * STAGE + 1024 * LPW * wave;
#pragma unroll
    for (int i = 0; i < LPW; ++i) {
      if (kin[i]) lds_dma16(p.kp + at, ko[i], to + 1024 * i);
      if (vin[i]) lds_dma16(p.vp + at, vo[i], to + TENSOR + 1024 * i);
    }
  };
  const int t0 = k0 / kPage, t1 = (k1 + kPage - 1) / kPage;
  int next = 0;
  if (t0 < t1) {
    issue(__builtin_amdgcn_readfirstlane(trow[t0]), 0);
    if (t0 + 1 < t1) next = __builtin_amdgcn_readfirstlane(trow[t0 + 1]);
  }
  u32x4 qf[MT][NKS];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int r = r0 + 32 * mt + n32;
    const bool live = r < all;
    const int qi = live ? r / p.G : 0;
    lim[mt] = live ? limit(qi) : 0;
    const uint16_t* qr = p.q + static_cast<int64_t>(it.q0 + qi) * p.q_st + static_cast<int64_t>(kvh * p.G + (live ? r - qi * p.G : 0)) * p.q_sh;
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) {
      const int c = 16 * ks + 8 * h;
      qf[mt][ks] = live && c < D ? *reinterpret_cast<const u32x4*>(qr + c) : u32x4{0, 0, 0, 0};
    }
  }
  f32x16 acc[MT][NCB];
  float m[MT], l[MT];  // of row n32: the running maximum (raw scores), the sum over this half's keys
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    m[mt] = kNegBig;
    l[mt] = 0.0f;
#pragma unroll
    for (int cb = 0; cb < NCB; ++cb)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[mt][cb][i] = 0.0f;
  }
  const float sl2 = p.scale_log2;

  for (int t = t0; t < t1; ++t) {
    const int buf = (t - t0) & 1;
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));  // this wave's share of page t
    __syncthreads();                           // everyone's; and page t - 1 is done with
    uint8_t* const kt = lds + buf * STAGE;
    uint8_t* const vt = kt + TENSOR;
    const int key = t * kPage, cnt = it.len - key;
    if (cnt < kPage) {  // rows that hold no token: whatever stands there must not count
      for (int i = threadIdx.x; i < (kPage - cnt) * UNITS; i += 64 * NW) *reinterpret_cast<u32x4*>(vt + 16 * (cnt * UNITS + i)) = u32x4{0, 0, 0, 0};
      __syncthreads();
    }
    if (t + 1 < t1) {
      issue(next, buf ^ 1);
      if (t + 2 < t1) next = __builtin_amdgcn_readfirstlane(trow[t + 2]);
    }
    if (key >= whi) continue;
    f32x16 s[MT][2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[mt][kb][i] = 0.0f;
      const int row = 32 * kb + n32;
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks) {
        const u32x4 a = *reinterpret_cast<const u32x4*>(kt + row * DP * 2 + 16 * wide_k_unit<DP>(row, 2 * ks + h));
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) s[mt][kb] = mfma32<BF>(a, qf[mt][ks], s[mt][kb]);
      }
    }
    u32x4 pa[MT][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      if (key + kPage > wlo) {
        const int left = lim[mt] - key;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (32 * kb + 8 * (i >> 2) + 4 * h + (i & 3) >= left) s[mt][kb][i] = -INFINITY;
      }
      auto probs = [&]() {
        const float nm = -m[mt] * sl2;
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            pa[mt][k][j] = pack2<BF>(__builtin_amdgcn_exp2f(fmaf(s[mt][k >> 1][8 * (k & 1) + 2 * j], sl2, nm)),
                                     __builtin_amdgcn_exp2f(fmaf(s[mt][k >> 1][8 * (k & 1) + 2 * j + 1], sl2, nm)));
      };
      probs();
      // 16-bit patterns of the non-negative probabilities order as their values do
      const u16x8 pm = __builtin_elementwise_max(
          __builtin_elementwise_max(__builtin_bit_cast(u16x8, pa[mt][0]), __builtin_bit_cast(u16x8, pa[mt][1])),
          __builtin_elementwise_max(__builtin_bit_cast(u16x8, pa[mt][2]), __builtin_bit_cast(u16x8, pa[mt][3])));
      const auto p2 = __builtin_elementwise_max(__builtin_elementwise_max(pm.s01, pm.s23), __builtin_elementwise_max(pm.s45, pm.s67));
      constexpr uint16_t kOver = BF ? 0x4380 : 0x5C00;  // 2^8
      if (__builtin_amdgcn_ballot_w64(p2.x > kOver || p2.y > kOver) != 0) {
        float mx = kNegBig;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int i = 0; i < 16; i += 2) mx = fmaxf(mx, fmaxf(s[mt][kb][i], s[mt][kb][i + 1]));
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float mn = fmaxf(m[mt], mx);
        const float alpha = __builtin_amdgcn_exp2f((m[mt] - mn) * sl2);
        m[mt] = mn;
        l[mt] *= alpha;
#pragma unroll
        for (int cb = 0; cb < NCB; ++cb)
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[mt][cb][i] *= alpha;
        probs();
      }
      float ps = 0.0f;
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t w = pa[mt][k][j];  // (a bit cast of a vector's element itself takes element 0)
          if constexpr (BF)
            ps = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w), (bf16x2{static_cast<__bf16>(1.0f), static_cast<__bf16>(1.0f)}), ps, false);
          else
            ps = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, w), (f16x2{static_cast<_Float16>(1.0f), static_cast<_Float16>(1.0f)}), ps, false);
        }
      l[mt] += ps;
    }
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
#pragma unroll
      for (int cb = 0; cb < NCB; ++cb) {
        // lane points at key 16 ks + 4 h + (l16 >> 2) (+ 8), channels 32 cb + 16 ((lane >> 4) & 1) + 4 (l16 & 3)
        const int row = 16 * ks + 4 * h + ((lane & 15) >> 2), u = 4 * cb + 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1);
        const uint8_t* at = vt + row * DP * 2 + 16 * wide_v_unit<DP>(row, u) + 8 * (lane & 1);
        const i16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_i16x4*>((lds_u8*)const_cast<uint8_t*>(at)));
        const i16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            reinterpret_cast<lds_i16x4*>((lds_u8*)const_cast<uint8_t*>(at + 8 * DP * 2)));  // (row + 8: the same exchange)
        const u32x2 w0 = __builtin_bit_cast(u32x2, v0), w1 = __builtin_bit_cast(u32x2, v1);
        const u32x4 a = {w0.x, w0.y, w1.x, w1.y};
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) acc[mt][cb] = mfma32<BF>(a, pa[mt][ks], acc[mt][cb]);
      }
    }
  }

  // ---- lane (n, h): row n, channels 32 cb + 8 q + 4 h .. + 3 ----
  const bool part = it.splits > 1;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const float lt = l[mt] + __shfl_xor(l[mt], 32, 64);
    const int r = r0 + 32 * mt + n32;
    if (r >= all) continue;
    if (part) {
      const int64_t pr = static_cast<int64_t>(blockIdx.x) * M + 32 * (MT * wave + mt) + n32;
      if (h == 0) p.part_ml[pr] = make_float2(m[mt] * sl2, lt);
#pragma unroll
      for (int cb = 0; cb < NCB; ++cb)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int c = 32 * cb + 8 * q + 4 * h;
          if (c < D) *reinterpret_cast<f32x4*>(p.part_o + pr * D + c) = f32x4{acc[mt][cb][4 * q], acc[mt][cb][4 * q + 1], acc[mt][cb][4 * q + 2], acc[mt][cb][4 * q + 3]};
        }
    } else {
      const int qi = r / p.G;
      const float inv = lt == 0.0f ? 0.0f : 1.0f / lt;  // no visible key: zeros
      uint16_t* dst = p.out + static_cast<int64_t>(it.q0 + qi) * p.o_st + static_cast<int64_t>(kvh * p.G + r - qi * p.G) * p.o_sh;
#pragma unroll
      for (int cb = 0; cb < NCB; ++cb)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int c = 32 * cb + 8 * q + 4 * h;
          u32x2 w;
          w.x = pack2<BF>(acc[mt][cb][4 * q] * inv, acc[mt][cb][4 * q + 1] * inv);
          w.y = pack2<BF>(acc[mt][cb][4 * q + 2] * inv, acc[mt][cb][4 * q + 3] * inv);
          if (c < D) *reinterpret_cast<u32x2*>(dst + c) = w;
        }
    }
  }
}

// The splits of a tile's rows joined in split order: D / 4 threads per row.
template <int M, bool BF>
__global__ __launch_bounds__(kThreads) void paged_merge_kernel(Params p) {
  const int kvh = blockIdx.x % p.Hkv;
  Item it;
  if (!find_item<M, true>(p, blockIdx.x / p.Hkv, it) || it.splits < 2) return;
  const int tpr = p.D / 4, rpb = kThreads / tpr;
  const int row = blockIdx.y * rpb + threadIdx.x / tpr, c = 4 * (threadIdx.x % tpr);
  const int rows = it.n * p.G - it.tile * M < M ? it.n * p.G - it.tile * M : M;
  if (threadIdx.x >= static_cast<unsigned>(rpb * tpr) || row >= rows) return;
  const int64_t item = it.first + static_cast<int64_t>(it.tiles - 1 - it.tile) * it.splits;
  if (item + it.splits > p.items) return;  // (counts that contradict each other)
  auto at = [&](int s) { return ((item + s) * p.Hkv + kvh) * M + row; };
  float mx = -INFINITY;
#pragma unroll 4
  for (int s = 0; s < it.splits; ++s) mx = fmaxf(mx, p.part_ml[at(s)].x);
  const float ms = mx == -INFINITY ? 0.0f : mx;
  float sum = 0.0f;
  f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (int s = 0; s < it.splits; ++s) {
    const float2 w = p.part_ml[at(s)];
    const f32x4 a = *reinterpret_cast<const f32x4*>(p.part_o + at(s) * p.D + c);
    const float f = __builtin_amdgcn_exp2f(w.x - ms);
    sum += w.y * f;
    o += a * f;
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  const int r = it.tile * M + row, qi = r / p.G;
  uint16_t* dst = p.out + static_cast<int64_t>(it.q0 + qi) * p.o_st + static_cast<int64_t>(kvh * p.G + r - qi * p.G) * p.o_sh + c;
#pragma unroll
  for (int i = 0; i < 4; ++i) dst[i] = f2w<BF>(o[i] * inv);
}

bool aligned16(const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15) == 0; }

// How one kernel's work of a call is cut, from the sizes the host knows.
struct Plan {
  int M = 0;              // matrix rows of a tile; 0: not launched
  int rows_of = kAll;
  int target = 0, least = 0;
  int64_t tiles = 0, items = 0;  // bounds: tiles of rows, items (per kv head)
};
struct Plans {
  Plan few, wide;
};

template <int DP>
struct Wide {  // waves and blocks of 32 rows per wave
  static constexpr int NW = DP > 128 ? 4 : 8, MT = 1, M = 32 * NW * MT;
};
int wide_rows(int D) { return D > 128 ? Wide<256>::M : Wide<128>::M; }

void bound_items(const Params& p, Plan& pl, int64_t tiles, int64_t pieces, int least) {
  pl.tiles = tiles;
  pl.target = static_cast<int>(cdiv(pieces, p.Hkv));
  pl.least = least;
  if (p.ppr * kPage <= least) pl.target = 0;
  pl.items = pl.tiles + pl.target;
}

int plan_of(const fade_paged_attn_args* a, Params& p, Plans& pl) {
  const char* what = "fade_paged_attn";
  if (a == nullptr) return einval("%s: null args", what);
  if (a->D < 8 || a->D > 256 || a->D % 8)
    return einval("%s: head_dim must be a multiple of 8 in [8, 256], got %lld", what, (long long)a->D);
  if (a->B < 1 || a->T < 0 || a->Hq < 1 || a->Hkv < 1 || a->n_pages < 1 || a->pages_per_row < 1)
    return einval("%s: B, Hq, Hkv, n_pages and pages_per_row must be positive, T not negative", what);
  if (a->Hq % a->Hkv) return einval("%s: needs Hq %% Hkv == 0 (got %lld/%lld)", what, (long long)a->Hq, (long long)a->Hkv);
  if (a->B > (1 << 20) || a->T > (1 << 24) || a->Hq > 65535 || a->T * (a->Hq / a->Hkv) >= (1ll << 31) ||
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
  p = Params{};
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
  // to the wide one; a call of at most 16 matrix rows per row on average is taken to
  // be a decoding step, all of it the few-row kernel's.
  const int64_t rows = p.T * p.G, live = p.B < p.T ? p.B : p.T;
  const bool step = rows <= kRows * p.B;
  pl.few.M = kRows;
  pl.few.rows_of = step ? kAll : kFew;
  // sum_b ceil(n_b G / M) <= T G / M + (rows with new tokens); two workgroups' worth of work per CU, in pieces of 256 keys or more
  bound_items(p, pl.few, step ? rows / kRows + live : live, 2 * num_cus(), 256);
  if (!step) {
    pl.wide.M = wide_rows(p.D);
    pl.wide.rows_of = kMany;
    const int64_t tiles = rows / pl.wide.M + live;
    // no splits where whole tiles fill the chip several times over
    bound_items(p, pl.wide, tiles, rows / pl.wide.M * p.Hkv >= 8 * num_cus() ? 0 : 2 * num_cus(), 512);
  }
  for (const Plan* k : {&pl.few, &pl.wide})
    if (k->items * p.Hkv >= (1ll << 24)) return einval("%s: shape too large (%lld items of work)", what, (long long)(k->items * p.Hkv));
  return FADE_OK;
}

int64_t part_rows(const Params& p, const Plan& pl) { return pl.target == 0 ? 0 : pl.items * p.Hkv * pl.M; }
// (the kernels run one after the other: their sums lie in the same memory)
int64_t part_rows(const Params& p, const Plans& pl) {
  const int64_t a = part_rows(p, pl.few), b = part_rows(p, pl.wide);
  return a > b ? a : b;
}
int64_t part_bytes(const Params& p, const Plans& pl) { return part_rows(p, pl) * (p.D * 4 + static_cast<int64_t>(sizeof(float2))); }

void apply(Params& p, const Plan& pl) {
  p.rows_of = pl.rows_of;
  p.target = pl.target;
  p.least = pl.least;
  p.per_item = pl.target > 0 ? 1.00002f / static_cast<float>(pl.target) : 0.0f;
  p.items = static_cast<uint32_t>(pl.items);
}

template <int M, bool BF>
int merge(const Params& p, const Plan& pl, hipStream_t st) {
  if (pl.target == 0) return FADE_OK;
  const dim3 grid(static_cast<unsigned>(p.Hkv * pl.tiles), static_cast<unsigned>(cdiv(M, kThreads / (p.D / 4))));
  hipLaunchKernelGGL((paged_merge_kernel<M, BF>), grid, dim3(kThreads), 0, st, p);
  return check_launch("fade_paged_attn (merge)");
}

template <int DP, bool BF>
int launch(Params& p, const Plans& pl, hipStream_t st) {
  apply(p, pl.few);
  hipLaunchKernelGGL((paged_few_kernel<DP, BF>), dim3(static_cast<unsigned>(p.Hkv * pl.few.items)), dim3(64 * Few<DP>::kWaves), 0, st, p);
  int rc = check_launch("fade_paged_attn");
  if (!rc) rc = merge<kRows, BF>(p, pl.few, st);
  if (rc || pl.wide.M == 0) return rc;
  typedef Wide<DP> W;
  apply(p, pl.wide);
  p.zero_tail = 0;
  hipLaunchKernelGGL((paged_wide_kernel<DP, W::NW, W::MT, BF>), dim3(static_cast<unsigned>(p.Hkv * pl.wide.items)), dim3(64 * W::NW), 0, st, p);
  rc = check_launch("fade_paged_attn");
  return rc ? rc : merge<W::M, BF>(p, pl.wide, st);
}

template <bool BF>
int launch_any(Params& p, const Plans& pl, void* stream) {
  hipStream_t st = as_stream(stream);
  if (p.D <= 64) return launch<64, BF>(p, pl, st);
  if (p.D <= 128) return launch<128, BF>(p, pl, st);
  return launch<256, BF>(p, pl, st);
}

}  // namespace
}  // namespace paged
}  // namespace fade

using namespace fade;
using namespace fade::paged;

FADE_API int fade_paged_attn_workspace_bytes(const fade_paged_attn_args* a, int64_t* bytes) {
  if (bytes == nullptr) return einval("fade_paged_attn_workspace_bytes: null output");
  Params p;
  Plans pl;
  const int rc = plan_of(a, p, pl);
  if (rc) return rc;
  *bytes = part_bytes(p, pl);
  return FADE_OK;
}

FADE_API int fade_paged_attn(const fade_paged_attn_args* a, void* workspace, int64_t workspace_bytes, void* stream) {
  Params p;
  Plans pl;
  const int rc = plan_of(a, p, pl);
  if (rc) return rc;
  if (p.T == 0) return FADE_OK;
  const int64_t need = part_bytes(p, pl);
  if (need > 0) {
    if (workspace == nullptr || workspace_bytes < need || !aligned16(workspace))
      return einval("fade_paged_attn: needs a 16-byte aligned workspace of %lld bytes", (long long)need);
    p.part_o = static_cast<float*>(workspace);
    p.part_ml = reinterpret_cast<float2*>(p.part_o + part_rows(p, pl) * p.D);
  }
  return a->dtype == FADE_DTYPE_BF16 ? launch_any<true>(p, pl, stream) : launch_any<false>(p, pl, stream);
}
