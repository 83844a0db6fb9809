// Attention of many query rows straight over the paged 8-bit cache (layouts: pages.hpp): the rows of a chunk of a
// prompt (causal, the last row at the last token) or of other sequences (cross attention: every row sees every token),
// and pages that neighbouring sequences share in front once for the rows of all of them.
//
// A workgroup takes 128 rows of one KV head, (token, query head) pairs, token major: four wavefronts of 32 rows, the
// columns of the matrix products.  A unit of 64 tokens lies in LDS as 16-bit numbers, which the codes turn to exactly: keys
// token major, values channel major, as their pages are.  S^T = K Q^T, the softmax in base 2 with one running reference
// and sum per column, O^T += V^T P^T.  Row m = 8 a + 4 g + b of tile s of S^T is token 32 g + 16 s + 4 a + b, so that lane
// half g holds the scores of tokens 32 g .. 32 g + 31 in order, which is how it reads a channel of V: 16 bytes, 8 tokens.
// The key scale multiplies the scores, the value scale the weights; both are float32.
// Weights times scale are bfloat16 (a scale has float32's range): rounded once for bfloat16 outputs, half a step of the
// type; as a pair that keeps 16 bits for half ones.
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstring>
#include <type_traits>
#include <vector>

#include "mfma_common.hpp"
#include "pages.hpp"

namespace kvq {
namespace {

constexpr int kThreads = 256, kTileRows = 128, kItemWords = 12, kMergeWords = 8, kSlots = 512, kMinPart = 8;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

template <bool BF16>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (BF16) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_f16(as_half8(a), as_half8(b), c, 0, 0, 0);
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const f32x2 v = {a, b};
  if constexpr (BF16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
  else return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, half2v));
}

// What rounding a pair of weights leaves, in the same type
template <bool BF16>
__device__ __forceinline__ uint32_t rest2(float a, float b, uint32_t w) {
  if constexpr (BF16) return pack2<true>(a - __uint_as_float(w << 16), b - __uint_as_float(w & 0xffff0000u));
  else return pack2<false>(a - h2f(w, 0), b - h2f(w, 1));
}

// Four codes as two pairs of numbers of the 16-bit type: exact.
template <int CODE, bool BF16>
__device__ __forceinline__ void widen4(uint32_t w, uint32_t& a, uint32_t& b) {
  if constexpr (CODE == kCodeE4M3) {
    if constexpr (BF16) {
      a = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false));
      b = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true));
    } else {
      a = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
      b = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true));
    }
  } else if constexpr (BF16) {
    const int s = static_cast<int>(w);
    a = pack2<true>(static_cast<float>(static_cast<int8_t>(s)), static_cast<float>(static_cast<int8_t>(s >> 8)));
    b = pack2<true>(static_cast<float>(static_cast<int8_t>(s >> 16)), static_cast<float>(static_cast<int8_t>(s >> 24)));
  } else {
    // 0x6400 | u is the half 1024 + u; u = code + 128
    const uint32_t u = w ^ 0x80808080u;
    const half2v z = {static_cast<_Float16>(1152.0f), static_cast<_Float16>(1152.0f)};
    a = w2(h2(__builtin_amdgcn_perm(0x64646464u, u, 0x07010700u)) - z);
    b = w2(h2(__builtin_amdgcn_perm(0x64646464u, u, 0x07030702u)) - z);
  }
}

template <int CODE, bool BF16>
__device__ __forceinline__ u32x4 widen8(uint32_t x, uint32_t y) {
  uint32_t r[4];
  widen4<CODE, BF16>(x, r[0], r[1]);
  widen4<CODE, BF16>(y, r[2], r[3]);
  return u32x4{r[0], r[1], r[2], r[3]};
}

#define KVQ_INLINE __attribute__((always_inline))

// f of the constants I .. N - 1: indexes of registers have to be known before any loop is unrolled
template <int I, int N, class F>
__device__ __forceinline__ void each(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    each<I + 1, N>(f);
  }
}

// An item: rows of one tile over some units of a slot.  {first packed row, tokens, slot, first unit, end, tokens visible to the first
// token, step, tokens of the slot, open buffer, part or -1}
struct WideArgs {
  const uint16_t* q;
  int64_t q_st, q_sh;
  const int* items;
  const int* table;
  int64_t max_blocks;
  int H, rep;
  float scale;                                // |scaling| * log2(e)
  uint32_t sign;                              // of scaling, for both halves of a word of q
  const uint8_t *kc, *vc;
  const float* sc;
  const uint16_t *ko, *vo;
  uint16_t* out;                              // (rows, Hq, D)
  float* part;                                // (parts, H): 128 x D sums, then 128 x {reference, sum}
};

template <int D, int P, int CODE, bool BF16>
__global__ __launch_bounds__(kThreads, 2) void paged_wide_kernel(WideArgs a) {
  constexpr int kPieces = D / 8;              // 16-byte pieces of a token's keys in LDS
  constexpr int kChunks = 4 * D, kPer = kChunks / kThreads;         // 16-byte pieces of a unit's codes, of a thread
  constexpr uint32_t kInf = BF16 ? 0x7f80u : 0x7c00u;
  __shared__ __align__(16) uint16_t ks[kUnit * D], vs[D * kUnit];
  __shared__ int flag[2];
  const int* it = a.items + kItemWords * (blockIdx.x / a.H);
  const int h = blockIdx.x % a.H;
  const int row0 = it[0], toks = it[1], slot = it[2], u0 = it[3], u1 = it[4], vis0 = it[5], vis_step = it[6], len = it[7], buf = it[8], piece = it[9];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 31, g = lane >> 5;
  const int full = len / P * P, u_full = (full + kUnit - 1) / kUnit, last = full / P - 1;
  const int u_end = u1 < u_full ? u1 : u_full;

  const int row = wave * 32 + col, tok = row / a.rep, hq = row % a.rep;
  const bool live = tok < toks;
  const int sees = vis0 + vis_step * tok, visible = !live ? 0 : sees < len ? sees : len;
  u32x4 q[D / 16];
  const uint32_t mask = live ? ~0u : 0u;
  const uint16_t* qp = a.q + (row0 + static_cast<int64_t>(live ? tok : 0)) * a.q_st + (static_cast<int64_t>(h) * a.rep + hq) * a.q_sh + 8 * g;
  each<0, D / 16>([&](auto i) { q[i.value] = (*reinterpret_cast<const u32x4*>(qp + 16 * i.value) ^ a.sign) & mask; });
  f32x16 o[D / 32], s[2];
  float m = -INFINITY, l = 0.0f;
  each<0, D / 32>([&](auto c) { each<0, 16>([&](auto e) { o[c.value][e.value] = 0.0f; }); });

  // Piece c of row r of keys lies at place c ^ k_swz(r) of its row, of values at c ^ v_swz(r): 16 lanes of a read meet 256
  // different bytes of the banks, and so do 16 of a write
  auto k_swz = [](int r) { return D == 128 ? (r & 7) | (r >> 5 & 1) << 3 : (r >> 1 & 3) | (r >> 5 & 1) << 2; };
  auto v_swz = [](int r) { return r >> 1 & 7; };
  auto k_put = [&](int r, int c, u32x4 w) KVQ_INLINE { *reinterpret_cast<u32x4*>(ks + r * D + (c ^ k_swz(r)) * 8) = w; };
  auto v_put = [&](int r, int c, u32x4 w) KVQ_INLINE { *reinterpret_cast<u32x4*>(vs + r * kUnit + (c ^ v_swz(r)) * 8) = w; };
  const int k_tok = 32 * (col >> 2 & 1) + 4 * (col >> 3) + (col & 3);
  auto read_k = [&](int i, int t) KVQ_INLINE {                      // channels 16 i + 8 g .., tile t
    const int r = k_tok + 16 * t;
    return *reinterpret_cast<const u32x4*>(ks + r * D + ((2 * i + g) ^ k_swz(r)) * 8);
  };
  auto read_v = [&](int c, int y) KVQ_INLINE {                      // channel 32 c + col, tokens 32 g + 8 y ..
    const int r = 32 * c + col;
    return *reinterpret_cast<const u32x4*>(vs + r * kUnit + ((4 * g + y) ^ v_swz(r)) * 8);
  };
  auto scores = [&]() KVQ_INLINE {
    each<0, 16>([&](auto e) { s[0][e.value] = s[1][e.value] = 0.0f; });
    each<0, D / 16>([&](auto i) { each<0, 2>([&](auto t) { s[t.value] = mfma32<BF16>(read_k(i.value, t.value), q[i.value], s[t.value]); }); });
  };
  // scores (register 16 t + e: token 32 g + 16 t + e of the unit) -> weights in s; o and l brought to the reference
  auto soft = [&](float scale, bool masked, int lim) KVQ_INLINE {
    if (masked)
      each<0, 32>([&](auto i) { s[i.value / 16][i.value % 16] = i.value < lim ? s[i.value / 16][i.value % 16] : -INFINITY; });
    float x = s[0][0];
    each<1, 32>([&](auto i) { x = fmaxf(x, s[i.value / 16][i.value % 16]); });
    // the reference moves only when a score passes it by 2^8: the accumulators are hardly ever scaled
    x = xmax32(x * scale);
    x = x > m + 8.0f ? x : m;
    const float safe = x == -INFINITY ? 0.0f : x, grow = __builtin_amdgcn_exp2f(m - safe);
    m = x;
    float sum = 0.0f;
    each<0, 32>([&](auto i) {
      const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i.value / 16][i.value % 16], scale, -safe));
      s[i.value / 16][i.value % 16] = p;
      sum += p;
    });
    l = l * grow + sum;
    if (__builtin_amdgcn_ballot_w64(grow != 1.0f)) each<0, D / 32>([&](auto c) { o[c.value] *= grow; });
  };

  const int* pages = a.table + slot * a.max_blocks;
  for (int u = u0; u < u_end; ++u) {
    const int t0 = u * kUnit;
    // the page of each half of the unit; half of the last one may lie behind the last page: masked
    const int b0 = t0 / P, b1 = (t0 + 32) / P < last ? (t0 + 32) / P : last;
    const int64_t p0 = static_cast<int64_t>(pages[b0]) * a.H + h, p1 = P == 32 ? static_cast<int64_t>(pages[b1]) * a.H + h : p0;
    u32x4 kw[kPer], vw[kPer];
    each<0, kPer>([&](auto i) {
      const int x = tid + i.value * kThreads, r = x / (D / 16), c = x % (D / 16), ch = x / 4, t = x % 4 * 16;
      kw[i.value] = *reinterpret_cast<const u32x4*>(a.kc + ((r < 32 ? p0 : p1) * P + ((t0 + r) & (P - 1))) * D + 16 * c);
      vw[i.value] = *reinterpret_cast<const u32x4*>(a.vc + ((t < 32 ? p0 : p1) * D + ch) * P + ((t0 + t) & (P - 1)));
    });
    const float2 z = reinterpret_cast<const float2*>(a.sc)[g ? p1 : p0];
    __syncthreads();
    each<0, kPer>([&](auto i) {
      const int x = tid + i.value * kThreads, r = x / (D / 16), c = x % (D / 16), ch = x / 4, t = x % 4;
      k_put(r, 2 * c, widen8<CODE, BF16>(kw[i.value][0], kw[i.value][1]));
      k_put(r, 2 * c + 1, widen8<CODE, BF16>(kw[i.value][2], kw[i.value][3]));
      v_put(ch, 2 * t, widen8<CODE, true>(vw[i.value][0], vw[i.value][1]));
      v_put(ch, 2 * t + 1, widen8<CODE, true>(vw[i.value][2], vw[i.value][3]));
    });
    __syncthreads();
    scores();
    // a block that a row sees nothing of may hold a NaN scale
    const int lim = (visible < full ? visible : full) - t0 - 32 * g;
    float kz = z.x * a.scale, vz = z.y;
    kz = kz < FLT_MIN ? FLT_MIN : kz;
    kz = lim > 0 ? kz : 1.0f;
    vz = lim > 0 ? vz : 0.0f;
    soft(kz, true, lim);
    each<0, 4>([&](auto y) {
      u32x4 hi, lo;
      each<0, 4>([&](auto e) {
        constexpr int at = y.value * 8 + 2 * e.value;
        const float p = s[at / 16][at % 16] * vz, r = s[at / 16][at % 16 + 1] * vz;
        hi[e.value] = pack2<true>(p, r);
        if constexpr (!BF16) lo[e.value] = rest2<true>(p, r, hi[e.value]);
      });
      each<0, D / 32>([&](auto c) {
        const u32x4 w = read_v(c.value, y.value);
        o[c.value] = mfma32<true>(w, hi, o[c.value]);
        if constexpr (!BF16) o[c.value] = mfma32<true>(w, lo, o[c.value]);
      });
    });
  }

  // Units of the open block
  const int64_t open = ((static_cast<int64_t>(slot) * 2 + buf) * a.H + h) * P * D;
  const uint16_t *ko = a.ko + open, *vo = a.vo + open;
  const int first_open = u0 > u_full ? u0 : u_full;
  for (int u = first_open; u < u1; ++u) {
    const int off = (u - u_full) * kUnit, t0 = full + off, rest = len - t0 < kUnit ? len - t0 : kUnit;
    __syncthreads();
    if (tid == 0) flag[u - u_full] = 0;
    for (int x = tid; x < kUnit * kPieces; x += kThreads) {
      const int r = x / kPieces, c = x % kPieces;
      u32x4 w = {0, 0, 0, 0};
      if (r < rest) w = *reinterpret_cast<const u32x4*>(ko + (off + r) * D + 8 * c);
      k_put(r, c, w);
    }
    __syncthreads();
    // what is hidden from a row may be an infinity or a NaN, and what lies behind the last token anything: such values go in as
    // zeros, and the rows that do see one have it afterwards
    for (int x = tid; x < D * 8; x += kThreads) {
      const int r = x / 8, c = x % 8;
      u32x4 w = {0, 0, 0, 0};
      bool bad = false;
      if (8 * c < rest) {
        w = *reinterpret_cast<const u32x4*>(vo + r * P + off + 8 * c);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool i0 = (w[e] & kInf) == kInf, i1 = (w[e] >> 16 & kInf) == kInf;
          bad |= i0 || i1;
          w[e] = (i0 ? 0u : w[e] & 0xffffu) | (i1 ? 0u : w[e] & 0xffff0000u);
        }
      }
      v_put(r, c, w);
      if (bad) flag[u - u_full] = 1;
    }
    __syncthreads();
    scores();
    soft(a.scale, true, visible - t0 - 32 * g);
    each<0, 4>([&](auto y) {
      u32x4 hi, lo;
      each<0, 4>([&](auto e) {
        constexpr int at = y.value * 8 + 2 * e.value;
        const float p = s[at / 16][at % 16], r = s[at / 16][at % 16 + 1];
        hi[e.value] = pack2<BF16>(p, r);
        if constexpr (!BF16) lo[e.value] = rest2<false>(p, r, hi[e.value]);
      });
      each<0, D / 32>([&](auto c) {
        const u32x4 w = read_v(c.value, y.value);
        o[c.value] = mfma32<BF16>(w, hi, o[c.value]);
        if constexpr (!BF16) o[c.value] = mfma32<false>(w, lo, o[c.value]);
      });
    });
  }
  // A visible value that is infinite or NaN is its channel's result, however small its weight
  for (int u = first_open; u < u1; ++u) {
    const int off = (u - u_full) * kUnit, t0 = full + off, rest = len - t0 < kUnit ? len - t0 : kUnit;
    if (!flag[u - u_full]) continue;
    for (int r = 0; r < rest; ++r)
      each<0, D / 32>([&](auto c) {
        each<0, 16>([&](auto e) {
          const uint16_t x = vo[(32 * c.value + 8 * (e.value / 4) + 4 * g + e.value % 4) * P + off + r];
          if (t0 + r < visible && (x & kInf) == kInf) o[c.value][e.value] += BF16 ? bf16_to_f32(x) : f16_to_f32(x);
        });
      });
  }

  l = xsum32(l);
  if (!live) return;
  if (piece >= 0) {
    float* part = a.part + (static_cast<int64_t>(piece) * a.H + h) * (kTileRows * (D + 2));
    each<0, D / 32>([&](auto c) {
      each<0, 4>([&](auto e) {
        const auto& x = o[c.value];
        *reinterpret_cast<float4*>(part + row * D + 32 * c.value + 8 * e.value + 4 * g) =
            make_float4(x[4 * e.value], x[4 * e.value + 1], x[4 * e.value + 2], x[4 * e.value + 3]);
      });
    });
    if (g == 0) *reinterpret_cast<float2*>(part + kTileRows * D + 2 * row) = make_float2(m, l);
    return;
  }
  const float inv = visible > 0 ? 1.0f / l : 0.0f;                  // a row that sees nothing: zeros
  uint16_t* out = a.out + ((row0 + static_cast<int64_t>(tok)) * a.H * a.rep + h * a.rep + hq) * D + 4 * g;
  each<0, D / 32>([&](auto c) {
    each<0, 4>([&](auto e) {
      const auto& x = o[c.value];
      *reinterpret_cast<uint2*>(out + 32 * c.value + 8 * e.value) =
          make_uint2(pack2<BF16>(x[4 * e.value] * inv, x[4 * e.value + 1] * inv), pack2<BF16>(x[4 * e.value + 2] * inv, x[4 * e.value + 3] * inv));
    });
  });
}

// One wavefront per row that is joined of several parts: those of its own tile and those of a tile of its shared front.
// merges[i] = {first packed row, tokens, first part, parts, token of the tile, the same of the front's tile}
template <int D, bool BF16>
__global__ __launch_bounds__(kThreads) void paged_wide_merge_kernel(WideArgs a, const int* __restrict__ merges) {
  const int* w = merges + kMergeWords * (blockIdx.x / a.H);
  const int h = blockIdx.x % a.H, lane = threadIdx.x & 63, row = blockIdx.y * (kThreads / 64) + (threadIdx.x >> 6);
  const int tok = row / a.rep, hq = row % a.rep;
  if (tok >= w[1]) return;
  constexpr int64_t kPart = kTileRows * (D + 2);
  const int64_t stride = a.H * kPart;
  float top = -INFINITY, l = 0.0f, o[D / 64] = {};
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const int first = w[2 + 3 * side], parts = w[3 + 3 * side], r = (w[4 + 3 * side] + tok) * a.rep + hq;
    const float* part = a.part + (static_cast<int64_t>(first) * a.H + h) * kPart;
    for (int i0 = 0; i0 < parts; i0 += 64) {
      const int i = i0 + lane;
      const float2 st = i < parts ? *reinterpret_cast<const float2*>(part + i * stride + kTileRows * D + 2 * r) : make_float2(-INFINITY, 0.0f);
      const float m = fmaxf(top, wave_max(st.x)), safe = m == -INFINITY ? 0.0f : m;
      const float old = __builtin_amdgcn_exp2f(top - safe), f = __builtin_amdgcn_exp2f(st.x - safe);
      l = l * old + wave_sum(f * st.y);
#pragma unroll
      for (int e = 0; e < D / 64; ++e) o[e] = weigh(old, o[e]);
      const int most = parts - i0 < 64 ? parts - i0 : 64;
      for (int k = 0; k < most; ++k) {
        const float fk = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f), k));
        const float* x = part + (i0 + k) * stride + r * D + lane * (D / 64);
#pragma unroll
        for (int e = 0; e < D / 64; ++e) o[e] += weigh(fk, x[e]);
      }
      top = m;
    }
  }
  const float inv = 1.0f / l;                 // a row that is joined sees a token at least
  uint16_t* out = a.out + ((w[0] + static_cast<int64_t>(tok)) * a.H * a.rep + h * a.rep + hq) * D + lane * (D / 64);
#pragma unroll
  for (int e = 0; e < D / 64; ++e) out[e] = BF16 ? f32_to_bf16(o[e] * inv) : f32_to_f16(o[e] * inv);
}


// ---- the plan (host) --------------------------------------------------------------------------

struct PlanItem {
  int32_t w[kItemWords];
};
struct PlanMerge {
  int32_t w[kMergeWords];
};
struct PlanWords {
  std::vector<PlanItem> items;
  std::vector<PlanMerge> merges;
  int64_t parts = 0;
};

// A tile of rows over the units [u0, u1) of a slot
struct Tile {
  int64_t row0, toks, slot, u0, u1, vis0, step, len, buf;
  int64_t front;                              // its front's first tile, or -1
  int64_t front_row0;                         // first packed row of that one
  bool joins, is_front;
  int64_t part, cut;
};

// A front pays for its joins from so many units of work on that it saves, per tile that is joined
constexpr int64_t kJoinUnits = 4;

int64_t units_before(int64_t tokens, int64_t len, int64_t page) {   // units of a slot that hold its first `tokens` tokens
  const int64_t full = len / page * page, u_full = (full + kUnit - 1) / kUnit;
  return tokens <= full ? (tokens + kUnit - 1) / kUnit : u_full + (tokens - full + kUnit - 1) / kUnit;
}

void plan_wide(const int64_t* lens, const int32_t* table, const uint8_t* open, int64_t max_blocks, int64_t page, const int64_t* seq,
               const int64_t* counts, int64_t n, int64_t rep, int64_t H, bool causal, PlanWords& out) {
  const int64_t per_tile = kTileRows / rep;   // tokens of a tile of rows
  struct Seq {
    int64_t slot, row0, count, len;
  };
  std::vector<Seq> some;
  int64_t row = 0;
  for (int64_t i = 0; i < n; ++i) {
    if (counts[i] > 0) {
      // rows that see all of one slot are one sequence's
      if (!causal && !some.empty() && some.back().slot == seq[i]) some.back().count += counts[i];
      else some.push_back({seq[i], row, counts[i], lens[seq[i]]});
    }
    row += counts[i];
  }
  auto tiles_of = [&](int64_t count) { return (count + per_tile - 1) / per_tile; };
  auto whole = [&](const Seq& s) { return (causal ? s.len - s.count : s.len) / page; };       // pages that all its rows see
  std::vector<Tile> tiles;
  for (size_t i = 0; i < some.size();) {
    size_t j = i + 1;
    int64_t common = 0, tokens = some[i].count, apart = tiles_of(some[i].count);
    for (; j < some.size(); ++j) {
      const int64_t a = whole(some[i]), b = whole(some[j]), most = a < b ? a : b;
      int64_t c = 0, cap = j > i + 1 && common < most ? common : most;
      while (c < cap && table[some[i].slot * max_blocks + c] == table[some[j].slot * max_blocks + c]) ++c;
      if (c * page < kUnit || 2 * c < common) break;
      common = c;
      tokens += some[j].count;
      apart += tiles_of(some[j].count);
    }
    int64_t front = j > i + 1 ? common * page / kUnit : 0;
    // with a front its tiles, and joins for all of them, instead of the front's units in every sequence's tiles
    if (front && (apart - tiles_of(tokens)) * front <= kJoinUnits * (apart + tiles_of(tokens))) front = 0;
    const int64_t first = static_cast<int64_t>(tiles.size());
    if (front)
      for (int64_t t = 0; t < tokens; t += per_tile)
        tiles.push_back({some[i].row0 + t, tokens - t < per_tile ? tokens - t : per_tile, some[i].slot, 0, front, front * kUnit, 0,
                         front * kUnit, 0, -1, 0, true, true, 0, 0});
    for (size_t b = i; b < j; ++b) {
      const Seq& s = some[b];
      for (int64_t t = 0; t < s.count; t += per_tile) {
        const int64_t toks = s.count - t < per_tile ? s.count - t : per_tile;
        const int64_t vis0 = causal ? s.len - s.count + t + 1 : s.len, seen = causal ? vis0 + toks - 1 : s.len;
        tiles.push_back({s.row0 + t, toks, s.slot, front, units_before(seen, s.len, page), vis0, causal ? 1 : 0, s.len, open[s.slot] & 1,
                         front ? first : -1, some[i].row0, front > 0, false, 0, 0});
      }
    }
    i = j;
  }
  // Where the tiles of rows do not fill kSlots places (two on each of 256 CUs), they are cut into the shortest parts that
  // fit: 8 units at least, which pay for the part's sums (64 KB)
  int64_t longest = 0;
  for (const Tile& t : tiles) longest = std::max(longest, t.u1 - t.u0);
  auto cut_of = [](const Tile& t, int64_t most) { return (t.u1 - t.u0 + most - 1) / most; };
  int64_t most = kMinPart, high = std::max<int64_t>(longest, kMinPart);
  if (static_cast<int64_t>(tiles.size()) * H > kSlots) most = high;
  while (most < high) {
    const int64_t mid = (most + high) / 2;
    int64_t count = 0;
    for (const Tile& t : tiles) count += std::max<int64_t>(cut_of(t, mid), 1);
    if (count * H <= kSlots) high = mid;
    else most = mid + 1;
  }
  for (Tile& t : tiles) {
    t.cut = cut_of(t, most);
    t.joins = t.joins || t.cut > 1;
    t.part = out.parts;
    if (t.joins) out.parts += t.cut;
    const int64_t count = t.joins ? t.cut : 1;
    for (int64_t c = 0; c < count; ++c) {
      const int64_t units = t.u1 - t.u0, a = t.u0 + units * c / count, b = t.u0 + units * (c + 1) / count;
      const int64_t w[kItemWords] = {t.row0, t.toks, t.slot, a, b, t.vis0, t.step, t.len, t.buf, t.joins ? t.part + c : -1, 0, 0};
      PlanItem it;
      for (int k = 0; k < kItemWords; ++k) it.w[k] = static_cast<int32_t>(w[k]);
      out.items.push_back(it);
    }
  }
  for (const Tile& t : tiles) {
    if (!t.joins || t.is_front) continue;
    for (int64_t a = 0; a < t.toks;) {
      int64_t toks = t.toks - a, w[kMergeWords] = {t.row0 + a, 0, t.part, t.cut, a, 0, 0, 0};
      if (t.front >= 0) {
        const int64_t at = t.row0 + a - t.front_row0, in = at % per_tile;
        const Tile& f = tiles[t.front + at / per_tile];
        toks = std::min(toks, per_tile - in);
        w[5] = f.part;
        w[6] = f.cut;
        w[7] = in;
      }
      w[1] = toks;
      PlanMerge m;
      for (int k = 0; k < kMergeWords; ++k) m.w[k] = static_cast<int32_t>(w[k]);
      out.merges.push_back(m);
      a += toks;
    }
  }
  // the longest first: the last workgroups to end are short ones
  std::sort(out.items.begin(), out.items.end(), [](const PlanItem& x, const PlanItem& y) {
    const int32_t a = x.w[4] - x.w[3], b = y.w[4] - y.w[3];
    return a != b ? a > b : x.w[0] != y.w[0] ? x.w[0] < y.w[0] : x.w[3] < y.w[3];
  });
}

}  // namespace
}  // namespace kvq

using namespace kvq;

extern "C" int kvq_paged_plan(const int64_t* lens, const int32_t* table, const uint8_t* open, int64_t slots, int64_t max_blocks, int64_t page,
                              const int64_t* seq, const int64_t* counts, int64_t n, int64_t rep, int64_t H, int causal, int32_t* words,
                              int64_t words_cap, int64_t* info) {
  KVQ_REQUIRE(lens && table && open && info && n >= 0 && (n == 0 || (seq && counts)), "kvq_paged_plan: null pointer");
  KVQ_REQUIRE(rep >= 1 && rep <= kTileRows && H >= 1 && (page == 32 || page == 64 || page == 128), "kvq_paged_plan: bad sizes");
  int64_t rows = 0;
  for (int64_t i = 0; i < n; ++i) {
    KVQ_REQUIRE(seq[i] >= 0 && seq[i] < slots, "kvq_paged_plan: no slot %lld (of %lld)", static_cast<long long>(seq[i]), static_cast<long long>(slots));
    KVQ_REQUIRE(counts[i] >= 0 && counts[i] < INT64_C(1) << 31, "kvq_paged_plan: counts must not be negative, and below 2^31");
    KVQ_REQUIRE(!causal || counts[i] <= lens[seq[i]], "kvq_paged_plan: slot %lld holds %lld tokens, %lld query rows are to be its last ones",
                static_cast<long long>(seq[i]), static_cast<long long>(lens[seq[i]]), static_cast<long long>(counts[i]));
    rows += counts[i];
    KVQ_REQUIRE(rows < INT64_C(1) << 31, "kvq_paged_plan: too many rows");
  }
  try {
    PlanWords p;
    plan_wide(lens, table, open, max_blocks, page, seq, counts, n, rep, H, causal != 0, p);
    info[0] = static_cast<int64_t>(p.items.size());
    info[1] = static_cast<int64_t>(p.merges.size());
    info[2] = p.parts;
    KVQ_REQUIRE(p.parts < INT64_C(1) << 31, "kvq_paged_plan: too many parts");
    if (!words || words_cap < kItemWords * info[0] + kMergeWords * info[1]) return KVQ_OK;
    memcpy(words, p.items.data(), sizeof(PlanItem) * p.items.size());
    memcpy(words + kItemWords * info[0], p.merges.data(), sizeof(PlanMerge) * p.merges.size());
  } catch (...) {
    KVQ_REQUIRE(false, "kvq_paged_plan: out of host memory");
  }
  return KVQ_OK;
}

extern "C" int64_t kvq_paged_attention_workspace(int64_t parts, int64_t H, int64_t D) {
  return parts < 0 || H < 1 || (D != 64 && D != 128) ? -1 : parts * H * kTileRows * (D + 2);
}

extern "C" int kvq_paged_attention(const void* q, int64_t q_st, int64_t q_sh, int dtype, int64_t Hq, int64_t H, int64_t D, float scaling,
                                   const int32_t* words, int64_t items, int64_t merges, int64_t parts, const int32_t* table,
                                   int64_t max_blocks, int64_t P, int code, const uint8_t* kc, const uint8_t* vc, const float* sc,
                                   const void* ko, const void* vo, void* out, float* workspace, int64_t workspace_floats, void* stream) {
  KVQ_REQUIRE(D == 64 || D == 128, "kvq_paged_attention: head_dim must be 64 or 128 (got %lld)", static_cast<long long>(D));
  KVQ_REQUIRE(P == 32 || P == 64 || P == 128, "kvq_paged_attention: pages hold 32, 64 or 128 tokens");
  KVQ_REQUIRE(dtype == KVQ_F16 || dtype == KVQ_BF16, "kvq_paged_attention: queries must be fp16 or bf16");
  KVQ_REQUIRE(code == kCodeInt8 || code == kCodeE4M3, "kvq_paged_attention: unknown code %d", code);
  KVQ_REQUIRE(H > 0 && Hq > 0 && Hq % H == 0 && Hq / H <= kTileRows && items >= 0 && merges >= 0 && parts >= 0, "kvq_paged_attention: bad sizes");
  if (items == 0) return KVQ_OK;
  KVQ_REQUIRE(q && words && table && kc && vc && sc && ko && vo && out && (workspace || !parts), "kvq_paged_attention: null pointer");
  KVQ_REQUIRE((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) % 16 == 0 &&
                  (q_st | q_sh) % 8 == 0,
              "kvq_paged_attention: rows and strides must be multiples of 16 bytes");
  KVQ_REQUIRE(items * H <= kMaxGrid && merges * H <= kMaxGrid, "kvq_paged_attention: too many rows");
  const int64_t need = kvq_paged_attention_workspace(parts, H, D);
  KVQ_REQUIRE(workspace_floats >= need || parts == 0, "kvq_paged_attention: workspace of %lld floats, %lld needed",
              static_cast<long long>(workspace_floats), static_cast<long long>(need));
  // a scaling of nothing would make a NaN of a hidden score's -inf: the smallest one, which makes zeros of the others
  const float scale = std::fabs(scaling) * 1.44269504088896341f;
  const WideArgs a{static_cast<const uint16_t*>(q), q_st, q_sh, words, table, max_blocks, static_cast<int>(H), static_cast<int>(Hq / H),
                   scale < FLT_MIN ? FLT_MIN : scale, std::signbit(scaling) ? 0x80008000u : 0u, kc, vc, sc,
                   static_cast<const uint16_t*>(ko), static_cast<const uint16_t*>(vo), static_cast<uint16_t*>(out), workspace};
  const dim3 grid(static_cast<uint32_t>(items * H)), joins(static_cast<uint32_t>(merges * H), kTileRows * 64 / kThreads);
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto run = [&](auto d, auto p, auto c, auto t) {
    constexpr int D_ = decltype(d)::value, P_ = decltype(p)::value, C_ = decltype(c)::value;
    constexpr bool T_ = decltype(t)::value;
    hipLaunchKernelGGL((paged_wide_kernel<D_, P_, C_, T_>), grid, dim3(kThreads), 0, s, a);
    if (merges) hipLaunchKernelGGL((paged_wide_merge_kernel<D_, T_>), joins, dim3(kThreads), 0, s, a, words + kItemWords * items);
  };
  auto by_type = [&](auto d, auto p, auto c) {
    if (dtype == KVQ_BF16) run(d, p, c, std::true_type{});
    else run(d, p, c, std::false_type{});
  };
  auto by_code = [&](auto d, auto p) {
    if (code == kCodeInt8) by_type(d, p, std::integral_constant<int, kCodeInt8>{});
    else by_type(d, p, std::integral_constant<int, kCodeE4M3>{});
  };
  auto by_page = [&](auto d) {
    if (P == 32) by_code(d, std::integral_constant<int, 32>{});
    else if (P == 64) by_code(d, std::integral_constant<int, 64>{});
    else by_code(d, std::integral_constant<int, 128>{});
  };
  if (D == 64) by_page(std::integral_constant<int, 64>{});
  else by_page(std::integral_constant<int, 128>{});
  KVQ_LAUNCH_CHECK("kvq_paged_attention");
  return KVQ_OK;
}
