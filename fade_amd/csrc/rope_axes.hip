// Rotary positions of several axes (time, height, width), and the append of
// rotated keys and of values to a paged cache.
//
// With r rotated channels of D, frequency i < r / 2 turns the channel pair
// (i, i + r / 2) of a token by the angle pos[axis(i)] * inv_freq_i:
//   y_i = x_i cos - x_{i + r/2} sin,   y_{i + r/2} = x_{i + r/2} cos + x_i sin
// and the channels past r stay as they are.  An angle is only needed modulo a
// full turn, so a frequency comes as a 64-bit fraction of a turn per position,
// round(inv_freq / (2 pi) * 2^64): position * fraction modulo 2^64 is one
// wrapping integer product, exact to 2^-65 of a turn per position (2^-34 at
// position 2^31), where a 32-bit float product has lost the angle long before.
// Its top 32 bits, as a float in [-1/2, 1/2) turns, go to the hardware's sine
// and cosine, which take turns (measured against 64 bits over 2^24 angles: 1.3e-7
// off at most; fp32 tensors use the library's sincospi).  The products are in
// fp32, rounded once.
//
// Bound by HBM: every row is read and written once.  A thread keeps one token's
// V = 16 bytes' worth of frequencies (their sines and cosines in registers) and
// walks the heads of its workgroup's tensor with them, so the trigonometry is paid
// once per workgroup's heads and a wave's access covers whole 128-byte runs of the
// rows: 16384 tokens of 40 heads (128 channels of 16 bits, 64 rotated on three
// axes) 72 to 76 us, 4.4 to 4.7 TB/s, where a large copy has 5.2; in fp32 126 us,
// 5.3 TB/s; 7900 tokens appended to their pages 44 us on new inputs, 32 on the same
// ones again (194 MB, partly in the last-level cache).  Calls of few tokens are bound
// by latency: no load waits for another one but for its address in the arguments (1187
// tokens of 32 heads 7.2 us, 32 tokens appended 4.1).
#include "fade_common.h"

namespace fade {
namespace {

constexpr int kThreads = 256;
constexpr int kPage = 64;

// Rows of one tensor [B, heads, S, D]: element strides, unit stride along D.
struct Rows {
  const void* src;
  void* dst;
  int64_t s_sb, s_sh, s_ss;
  int64_t d_sb, d_sh, d_ss;
};

struct RopeParams {
  int64_t tokens, S;  // B * S of them
  uint32_t first;     // this launch's first
  int D, half;        // channels of a row, rotated pairs
  int heads[3];       // of q, k, v (v only in an append)
  int first_group[3]; // of each tensor's heads in the grid's second dimension
  int heads_per_block;
  int inverse, append;
  const void* pos;    // axis a of token (b, s) at a * pos_sa + b * pos_sb + s * pos_ss
  int64_t pos_sa, pos_sb, pos_ss;
  int pos64, axes;
  Rows rows[3];       // append: k's and v's dst are pages [n_pages][Hkv][64][D]
  const int32_t* slots;
  int64_t n_pages;
  const uint64_t* turn;  // [half], in device memory: as arguments they cost 1 to 2 us a launch
  const uint8_t* axis;
};

// sine and cosine of an angle in turns
template <typename T>
__device__ __forceinline__ void sincos_turns(float t, float& s, float& c) {
  if constexpr (sizeof(T) == 4) {
    sincospif(2.0f * t, &s, &c);
  } else {
    s = __builtin_amdgcn_sinf(t);
    c = __builtin_amdgcn_cosf(t);
  }
}

template <typename T, int V>
struct alignas(V * sizeof(T)) Vec {
  T e[V];
};

// T: uint16_t (fp16 bits), Bf16 or float; V: channels per access.  A unit of
// work is 2 V channels of a row: pairs V u .. of the rotated halves, or the
// channels r + 2 V (u - half / V) .. past them.
template <typename T, int V>
__global__ __launch_bounds__(kThreads) void rope_kernel(RopeParams p) {
  typedef Vec<T, V> Vt;
  // a workgroup has heads of one tensor
  const int which = blockIdx.y >= static_cast<unsigned>(p.first_group[2]) ? 2 : (blockIdx.y >= static_cast<unsigned>(p.first_group[1]) ? 1 : 0);
  const Rows& r = p.rows[which];
  const unsigned units = static_cast<unsigned>(p.D) / (2 * V);
  const unsigned per_block = kThreads / units, lrow = threadIdx.x / units;
  const int u = static_cast<int>(threadIdx.x - lrow * units);
  const uint32_t t = p.first + blockIdx.x * per_block + lrow;  // (tokens < 2^31)
  if (lrow >= per_block || t >= static_cast<uint32_t>(p.tokens)) return;
  const uint32_t b = t / static_cast<uint32_t>(p.S), s = t - b * static_cast<uint32_t>(p.S);
  const int rot_units = p.half / V;
  const bool rot = u < rot_units;
  const int c0 = rot ? V * u : 2 * p.half + 2 * V * (u - rot_units);  // the unit's first channel
  const int c1 = rot ? c0 + p.half : c0 + V;                          // and the first of its other V

  const int h0 = (static_cast<int>(blockIdx.y) - p.first_group[which]) * p.heads_per_block;
  const int h1 = h0 + p.heads_per_block < p.heads[which] ? h0 + p.heads_per_block : p.heads[which];
  const bool paged = p.append && which > 0;
  const T* src = static_cast<const T*>(r.src) + b * r.s_sb + h0 * r.s_sh + s * r.s_ss;
  // the loads do not wait for one another: the first head's row, the slot, positions on every axis, the frequencies
  Vt x = *reinterpret_cast<const Vt*>(src + c0), y = *reinterpret_cast<const Vt*>(src + c1);
  int32_t slot = 0;
  if (paged) slot = p.slots[t];
  float sn[V], cs[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    sn[i] = 0.0f;
    cs[i] = 1.0f;
  }
  if (p.pos != nullptr && which < 2) {
    const int64_t at = b * p.pos_sb + s * p.pos_ss;
    int64_t pos[FADE_ROPE_MAX_AXES];
    if (p.pos64) {
#pragma unroll
      for (int k = 0; k < FADE_ROPE_MAX_AXES; ++k) pos[k] = static_cast<const int64_t*>(p.pos)[at + (k < p.axes ? k : 0) * p.pos_sa];
    } else {
#pragma unroll
      for (int k = 0; k < FADE_ROPE_MAX_AXES; ++k) pos[k] = static_cast<const int32_t*>(p.pos)[at + (k < p.axes ? k : 0) * p.pos_sa];
    }
    const int f0 = rot ? c0 : 0;
    uint64_t turn[V];
    uint32_t ax[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      turn[i] = p.turn[f0 + i];
      ax[i] = p.axis[f0 + i];
    }
    const float sign = p.inverse ? -1.0f : 1.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      int64_t ps = pos[0];
#pragma unroll
      for (int k = 1; k < FADE_ROPE_MAX_AXES; ++k) ps = ax[i] == k ? pos[k] : ps;
      const uint64_t a = static_cast<uint64_t>(ps) * turn[i];
      sincos_turns<T>(static_cast<float>(static_cast<int32_t>(a >> 32)) * 0x1p-32f, sn[i], cs[i]);
      sn[i] *= sign;
    }
  }
  T* dst = static_cast<T*>(r.dst);
  int64_t d_sh = r.d_sh;
  if (paged) {
    const int32_t page = slot / kPage, off = slot % kPage;
    if (slot < kPage || page >= p.n_pages) return;  // no place (page 0 holds no tokens)
    d_sh = static_cast<int64_t>(kPage) * p.D;
    dst += (static_cast<int64_t>(page) * p.heads[which] + h0) * d_sh + off * p.D;
  } else {
    dst += b * r.d_sb + h0 * d_sh + s * r.d_ss;
  }
  for (int hh = h0; hh < h1; ++hh) {
    Vt a = x, c = y;
    if (hh + 1 < h1) {  // the next head's row
      src += r.s_sh;
      x = *reinterpret_cast<const Vt*>(src + c0);
      y = *reinterpret_cast<const Vt*>(src + c1);
    }
    if (rot && which < 2) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float xf = to_f32(a.e[e]), yf = to_f32(c.e[e]);
        // (as they stand: the same operations in every instance)
        float lo = __fmaf_rn(xf, cs[e], -__fmul_rn(yf, sn[e])), hi = __fmaf_rn(yf, cs[e], __fmul_rn(xf, sn[e]));
        asm("" : "+v"(lo), "+v"(hi));  // (fp32 sums: the compiler joins some with their rounding to fp16, others not)
        a.e[e] = from_f32<T>(lo);
        c.e[e] = from_f32<T>(hi);
      }
    }
    *reinterpret_cast<Vt*>(dst + c0) = a;
    *reinterpret_cast<Vt*>(dst + c1) = c;
    dst += d_sh;
  }
}

template <typename T>
int rope_launch(RopeParams& p, bool wide, void* stream) {
  constexpr int V = 16 / static_cast<int>(sizeof(T));
  const int units = p.D / (2 * (wide ? V : 1));
  const int64_t bx = cdiv(p.tokens, kThreads / units);
  const int all = p.heads[0] + p.heads[1] + p.heads[2];
  // heads are spread over workgroups while there are fewer than two per CU (one, two, four per CU: 16384 tokens x 40
  // heads 71.6, 71.5, 73.3 us; 1187 x 32 7.9, 7.5, 8.0; 7900 tokens appended 39.6, 36.8, 37.2)
  int split = 1;
  while (bx * split < 2 * num_cus() && split < all) split *= 2;
  p.heads_per_block = static_cast<int>(cdiv(all, split));
  int groups = 0;
  for (int i = 0; i < 3; ++i) {
    p.first_group[i] = groups;
    groups += static_cast<int>(cdiv(p.heads[i], p.heads_per_block));
  }
  // (a launch has fewer than 2^32 threads along x)
  const int64_t most = ((1ll << 32) / kThreads) - 1;
  for (int64_t b0 = 0; b0 < bx; b0 += most) {
    p.first = static_cast<uint32_t>(b0 * (kThreads / units));
    const dim3 grid(static_cast<unsigned>(bx - b0 < most ? bx - b0 : most), static_cast<unsigned>(groups));
    if (wide) hipLaunchKernelGGL((rope_kernel<T, V>), grid, dim3(kThreads), 0, as_stream(stream), p);
    else hipLaunchKernelGGL((rope_kernel<T, 1>), grid, dim3(kThreads), 0, as_stream(stream), p);
    const int rc = check_launch("fade_rope_axes");
    if (rc) return rc;
  }
  return FADE_OK;
}

int rope_any(const fade_rope_args* a, bool append, const char* what, void* stream) {
  if (a == nullptr) return einval("%s: null args", what);
  if (a->dtype != FADE_DTYPE_F16 && a->dtype != FADE_DTYPE_BF16 && (append || a->dtype != FADE_DTYPE_F32))
    return einval("%s: unknown dtype %d", what, a->dtype);
  if (a->D < 2 || a->D > 2 * FADE_ROPE_MAX_FREQS || a->D % 2) return einval("%s: head_dim must be even, 2 to 256, got %lld", what, (long long)a->D);
  if (a->n_axes < 1 || a->n_axes > FADE_ROPE_MAX_AXES) return einval("%s: 1 to %d axes, got %d", what, FADE_ROPE_MAX_AXES, a->n_axes);
  if (a->n_freqs < 0 || 2 * a->n_freqs > a->D) return einval("%s: %lld frequencies for head_dim %lld", what, (long long)a->n_freqs, (long long)a->D);
  if (a->B < 0 || a->S < 0 || a->Hq < 0 || a->Hkv < 0 || a->Hq > 65535 || a->Hkv > 65535) return einval("%s: bad shape", what);
  if (append && a->B > 1) return einval("%s: tokens come as one row", what);
  if (a->S != 0 && a->B >= (1ll << 31) / a->S) return einval("%s: shape too large", what);
  const int64_t tokens = a->B * a->S;
  if (tokens == 0 || a->Hq + a->Hkv == 0) return FADE_OK;
  if ((a->Hq > 0 && (!a->q.src || !a->q.dst)) || (a->Hkv > 0 && (!a->k.src || !a->k.dst))) return einval("%s: null q or k", what);
  if (append && (!a->slots || (a->Hkv > 0 && (!a->v.src || !a->v.dst)) || a->n_pages < 1 || a->n_pages >= (1ll << 31) / kPage))
    return einval("%s: null v or slots, or a bad number of pages", what);
  if (!append && a->n_freqs > 0 && a->positions == nullptr) return einval("%s: null positions", what);
  RopeParams p{};
  p.tokens = tokens;
  p.S = a->S;
  p.D = static_cast<int>(a->D);
  p.half = static_cast<int>(a->n_freqs);
  p.heads[0] = static_cast<int>(a->Hq);
  p.heads[1] = static_cast<int>(a->Hkv);
  p.heads[2] = append ? p.heads[1] : 0;
  p.inverse = a->inverse;
  p.append = append;
  p.pos = p.half > 0 ? a->positions : nullptr;
  p.pos_sa = a->pos_sa;
  p.pos_sb = a->pos_sb;
  p.pos_ss = a->pos_ss;
  p.pos64 = a->pos64;
  p.axes = a->n_axes;
  p.slots = a->slots;
  p.n_pages = a->n_pages;
  if (p.half > 0 && p.pos != nullptr && (!a->turn || !a->axis)) return einval("%s: null turn or axis", what);
  p.turn = a->turn;
  p.axis = a->axis;
  // 16-byte accesses: whole units of both halves and aligned rows
  const int V = a->dtype == FADE_DTYPE_F32 ? 4 : 8, size = 16 / V;
  bool wide = p.D % (2 * V) == 0 && p.half % V == 0;
  auto rows = [&](const fade_rope_rows& x, bool paged) {
    Rows r{x.src, x.dst, x.src_sb, x.src_sh, x.src_ss, x.dst_sb, x.dst_sh, x.dst_ss};
    uintptr_t m = reinterpret_cast<uintptr_t>(x.src) | reinterpret_cast<uintptr_t>(x.dst);
    m |= static_cast<uintptr_t>((a->B > 1 ? r.s_sb : 0) | r.s_sh | r.s_ss) * size;
    if (!paged) m |= static_cast<uintptr_t>((a->B > 1 ? r.d_sb : 0) | r.d_sh | r.d_ss) * size;
    if (m % 16) wide = false;
    return r;
  };
  if (p.heads[0]) p.rows[0] = rows(a->q, false);
  if (p.heads[1]) p.rows[1] = rows(a->k, append);
  if (p.heads[2]) p.rows[2] = rows(a->v, append);
  if (a->dtype == FADE_DTYPE_F16) return rope_launch<uint16_t>(p, wide, stream);
  if (a->dtype == FADE_DTYPE_BF16) return rope_launch<Bf16>(p, wide, stream);
  return rope_launch<float>(p, wide, stream);
}

}  // namespace
}  // namespace fade

FADE_API int fade_rope_axes(const fade_rope_args* a, void* stream) { return fade::rope_any(a, false, "fade_rope_axes", stream); }

FADE_API int fade_paged_append(const fade_rope_args* a, void* stream) { return fade::rope_any(a, true, "fade_paged_append", stream); }
