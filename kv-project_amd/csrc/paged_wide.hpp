// Attention of many query rows straight over the paged 8-bit cache (layouts: pages.hpp): the rows of a chunk of a
// prompt (causal, the last row at the last token) or of other sequences (cross attention: every row sees every token),
// and pages that neighbouring sequences share in front once for the rows of all of them.
//
// A workgroup takes 128 rows of one KV head, (token, query head) pairs, token major: four wavefronts of 32 rows, the
// columns of the matrix products.  A unit of 64 tokens lies in LDS as 16-bit numbers, which the codes turn to exactly: keys
// token major, values channel major, as their pages are.  S^T = K Q^T, the softmax in base 2 with one running reference
// and sum per column, O^T += V^T P^T.  Row m = 8 a + 4 g + b of tile s of S^T is token 32 g + 16 s + 4 a + b, so that lane
// half g holds the scores of tokens 32 g .. 32 g + 31 in order, which is how it reads a channel of V: 16 bytes, 8 tokens.
// The key scale multiplies the scores, the value scale the weights; both are float32.  Weights times scale are rounded once to
// the inputs' type, half a step of the outputs'.  bfloat16 has a scale's range; for half types the accumulators are held in
// units of a power of two near the scale (a row's own: only blocks that it sees count), and the reference weighs 2^7: what a weight loses
// below 2^-14 is at most 2^-28 of its block's largest value, or with pages of 32 tokens of the larger one's of the two in a unit; the sum
// loses nothing of it.
//
// What bounds it: matrix cores and vector unit together.  A unit of 128 rows is 32 products of 32x32x16 a wavefront with head_dim 128
// (1024 cycles) beside 220 vector instructions, an exponential for 256 multiplications; two wavefronts to a SIMD fill each other's gaps,
// and reading the codes once for 128 or 256 rows leaves memory idle.  32 questions of 301 to 700 tokens behind 16384, 32 / 8 heads
// of 128, int8, bf16: 3700-4020 us by card, 1.03-1.12 PFLOP/s, matrix cores busy 54-56%, vector unit 54-59%, at 2.1 GHz of 2.4; four fp16
// chunks of 512 to 1531 tokens behind 9000, head_dim 64, e4m3: 346-382 us, 35% and 65%.  Four wavefronts at head_dim 128 spill 2 to 9 of
// their 256 registers.
#pragma once
#include <cfloat>
#include <type_traits>

#include "mfma_common.hpp"
#include "pages.hpp"

namespace kvq {

// An item: rows of one tile over some units of a slot.  {first packed row, tokens, slot, first unit, end, tokens visible to the first
// token, step, tokens of the slot, open buffer, part or -1}
// A join of rows: {first packed row, tokens, first part, parts, token of the tile, the same of the front's tile}
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
  float* part;                                // (parts, H): of each row of the tile D sums, then {reference, sum}
};

constexpr int kItemWords = 12, kMergeWords = 8;
constexpr int64_t kSpread = 12;               // parts of a row from which on a workgroup joins it

// The launches of one head_dim: the rows, then the joins
void launch_wide_64(const WideArgs& a, int page, int code, bool bf16, int waves, int64_t items, int64_t merges, int64_t most_parts, hipStream_t stream);
void launch_wide_128(const WideArgs& a, int page, int code, bool bf16, int waves, int64_t items, int64_t merges, int64_t most_parts, hipStream_t stream);

namespace {

constexpr int kThreads = 256;

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

// 16 bytes of device memory: said so, since an address that is put together in several steps is otherwise read as one that may
// be LDS, and waits for LDS then wait for it
__device__ __forceinline__ u32x4 load16(const void* p) {
  return *reinterpret_cast<const __attribute__((address_space(1))) u32x4*>(reinterpret_cast<uintptr_t>(p));
}

// f of the constants I .. N - 1: indexes of registers have to be known before any loop is unrolled
template <int I, int N, class F>
__device__ __forceinline__ void each(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    each<I + 1, N>(f);
  }
}

// Iteration j takes unit j of the codes through the softmax, beside matrix products that do not depend on it: O += V(j-1)
// P(j-1); then S(j+1) = K(j+1) Q, beside the widening of K(j+2) and V(j) from registers to LDS (two buffers each, one barrier an
// iteration), whose codes were fetched an iteration earlier.  The number of units is rounded up to an odd one, so that buffers
// and registers of even and odd ones have fixed places.  Units of the open block follow, one at a time.
template <int D, int P, int CODE, bool BF16, int W>
__global__ __launch_bounds__(64 * W, 2) void paged_wide_kernel(WideArgs a) {
  constexpr int kThreads = 64 * W, kTileRows = 32 * W;
  constexpr int kPieces = D / 8;              // 16-byte pieces of a token's keys in LDS
  constexpr int kPer = 4 * D / kThreads;      // 16-byte pieces of a unit's key codes of a thread, and of its value codes
  constexpr int kBuf = kUnit * D;
  constexpr uint32_t kInf = BF16 ? 0x7f80u : 0x7c00u;
  constexpr bool kOne = P >= kUnit;           // a unit lies in one page
  __shared__ __align__(16) uint16_t ks[2][kBuf], vs[2][kBuf];
  __shared__ int flag[2];
  const int* it = a.items + kItemWords * (blockIdx.x / a.H);
  const int h = blockIdx.x % a.H;
  const int row0 = it[0], toks = it[1], slot = it[2], u0 = it[3], u1 = it[4], vis0 = it[5], vis_step = it[6], len = it[7], buf = it[8], piece = it[9];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31, g = lane >> 5;
  const int full = len / P * P, u_full = (full + kUnit - 1) / kUnit, last = full / P - 1;
  const int u_end = u1 < u_full ? u1 : u_full;

  const int row = wave * 32 + col, tok = row / a.rep, hq = row % a.rep;
  const bool live = tok < toks;
  const int sees = vis0 + vis_step * tok, visible = !live ? 0 : sees < len ? sees : len;
  // every lane reads a row, dead ones the first
  u32x4 q[D / 16];
  const uint32_t mask = live ? ~0u : 0u;
  const uint16_t* qp = a.q + (row0 + static_cast<int64_t>(live ? tok : 0)) * a.q_st + (static_cast<int64_t>(h) * a.rep + hq) * a.q_sh + 8 * g;
  each<0, D / 16>([&](auto i) { q[i.value] = *reinterpret_cast<const u32x4*>(qp + 16 * i.value); });
  f32x16 o[D / 32], s[2][2];                  // s, p: of even and odd units
  u32x4 p[2][4];
  float m = -INFINITY, l = 0.0f, grow = 1.0f; // the exponents' reference, this lane's part of the sum, what o is to be scaled by
  each<0, D / 32>([&](auto c) { each<0, 16>([&](auto e) { o[c.value][e.value] = 0.0f; }); });

  // Piece c of row r of keys lies at place c ^ k_swz(r) of its row, of values at c ^ v_swz(r): 16 lanes of a read meet 256
  // different bytes of the banks, and 8 of a write 128: for that a thread takes the piece of its number with bits 2 and 3
  // exchanged
  const int tx = (tid & ~12) | (tid & 4) << 1 | (tid & 8) >> 1;
  auto k_swz = [](int r) { return D == 128 ? (r & 7) | (r >> 5 & 1) << 3 : (r >> 1 & 3) | (r >> 5 & 1) << 2; };
  auto v_swz = [](int r) { return r >> 1 & 7; };
  auto k_put = [&](int par, int r, int c, u32x4 w) KVQ_INLINE { *reinterpret_cast<u32x4*>(ks[par] + r * D + (c ^ k_swz(r)) * 8) = w; };
  auto v_put = [&](int par, int r, int c, u32x4 w) KVQ_INLINE { *reinterpret_cast<u32x4*>(vs[par] + r * kUnit + (c ^ v_swz(r)) * 8) = w; };
  const int k_tok = 32 * (col >> 2 & 1) + 4 * (col >> 3) + (col & 3), k_x = g ^ k_swz(k_tok), v_x = (4 * g) ^ v_swz(col);
  auto read_k = [&](auto par, int t) KVQ_INLINE {        // operand t of K: channels 16 (t / 2) + 8 g .., tile t % 2 (rows 16 apart have the
    return *reinterpret_cast<const u32x4*>(ks[decltype(par)::value] + (k_tok + 16 * (t % 2)) * D + ((2 * (t / 2)) ^ k_x) * 8);   // same swizzle)
  };
  auto read_v = [&](auto par, int t) KVQ_INLINE {        // operand t of V^T: channels 32 c + col, tokens 32 g + 8 y ..
    const int y = t / (D / 32), c = t % (D / 32);
    return *reinterpret_cast<const u32x4*>(vs[decltype(par)::value] + (32 * c + col) * kUnit + (y ^ v_x) * 8);
  };

  if (tid < 2) flag[tid] = 0;                 // a barrier later
  const int* pages = a.table + slot * a.max_blocks;
  const int units = u_end - u0, tiles = units > 0 ? units | 1 : 0;
  int whole = (vis0 < full ? vis0 : full) / kUnit - u0;             // units that every row sees whole
  whole = whole < 0 ? 0 : whole < units ? whole : units;
  // Codes of unit j, its pages a unit ahead of them.  (Behind the last unit: it again, masked; half of the last one may lie behind
  // the last page.)
  struct Ids {
    int a, b;                                 // of the unit's halves
  };
  auto unit_of = [&](int j) KVQ_INLINE { return u0 + (j < units ? j : units - 1); };
  auto ids_of = [&](int j) KVQ_INLINE {
    const int b0 = unit_of(j) * kUnit / P, b1 = b0 < last ? b0 + 1 : last;
    Ids r;
    r.a = pages[b0];
    r.b = kOne ? r.a : pages[b1];
    return r;
  };
  auto at_of = [&](int id) KVQ_INLINE { return static_cast<int64_t>(__builtin_amdgcn_readfirstlane(id)) * a.H + h; };
  u32x4 kw[kPer], vw[kPer];
  auto fetch_k = [&](Ids ids, int j, auto i) KVQ_INLINE {
    if constexpr (kOne) {
      const uint8_t* base = a.kc + at_of(ids.a) * (P * D) + (unit_of(j) * kUnit & (P - 1)) * D;
      kw[i.value] = load16(base + (tx + i.value * kThreads) * 16);
    } else if constexpr (kPer == 2) {         // a thread's pieces are of one half each
      kw[i.value] = load16(a.kc + at_of(i.value ? ids.b : ids.a) * (P * D) + tx * 16);
    } else {                                  // a wavefront's
      kw[i.value] = load16(a.kc + at_of(wave >= W / 2 ? ids.b : ids.a) * (P * D) + (tx & (kThreads / 2 - 1)) * 16);
    }
  };
  auto fetch_v = [&](Ids ids, int j, auto i) KVQ_INLINE {
    const int x = tx + i.value * kThreads, ch = x / 4, t = x % 4 * 16;
    if constexpr (kOne) {
      const uint8_t* base = a.vc + at_of(ids.a) * (P * D) + (unit_of(j) * kUnit & (P - 1));
      vw[i.value] = load16(base + ch * P + t);
    } else {
      const int64_t first = at_of(ids.a), second = at_of(ids.b), at = t < 32 ? first : second;
      vw[i.value] = load16(a.vc + at * (P * D) + ch * P + (t & 31));
    }
  };
  auto scales_of = [&](Ids ids) KVQ_INLINE {
    const int64_t first = at_of(ids.a), second = at_of(ids.b);        // not behind a branch, which would part the products' steps
    return reinterpret_cast<const float2*>(a.sc)[kOne || !g ? first : second];
  };
  // 8 codes of piece i / 2 each
  auto widen_k = [&](int par, auto i) KVQ_INLINE {
    const int x = tx + i.value / 2 * kThreads;
    const u32x4 w = kw[i.value / 2];
    k_put(par, x / (D / 16), 2 * (x % (D / 16)) + i.value % 2, widen8<CODE, BF16>(w[2 * (i.value % 2)], w[2 * (i.value % 2) + 1]));
  };
  auto widen_v = [&](int par, auto i) KVQ_INLINE {
    const int x = tx + i.value / 2 * kThreads;
    const u32x4 w = vw[i.value / 2];
    v_put(par, x / 4, 2 * (x % 4) + i.value % 2, widen8<CODE, BF16>(w[2 * (i.value % 2)], w[2 * (i.value % 2) + 1]));
  };

  // The softmax of a unit: share i is the weights 2 i, 2 i + 1 (register 16 t + e: token 32 g + 16 t + e).  The weights come
  // multiplied by the value scale, as its logarithm lr in the exponent, and their sum is divided by it once.  kz: what makes
  // exponents of scores.
  constexpr float kLift = BF16 ? 0.0f : 7.0f; // log2 of the reference's weight
  constexpr float kMost = BF16 ? 0x1p13f : 0x1p15f;
  constexpr float kWindow = BF16 ? 0x1p-60f : 0x1p-4f;              // a scale in its unit, unless it shares that with a larger one
  float base = 0.0f, safe, sum, kz, lr, inv_r, wx, wz;
  float unit = 0.0f;                          // a power of two near the value scales that the row has met: o is held in units of it; 0: none yet
  // The reference from the unit's scores, where one passes it by more than 2^slack.  lim: how many of this lane's 32 tokens the row
  // sees.  Only units that some row does not see whole look for it: in the others the weights are taken by the one there is, and
  // where a lane's come to more than kMost, taken again.  Weights of up to that cost no accuracy, and a maximum of every unit costs 30 of
  // its 207 vector instructions with head_dim 64, in a row before the first weight (four fp16 chunks 398 -> 376 us; 32 questions
  // behind 16384, head_dim 128, 3925 -> 3777).
  auto find = [&](auto par, bool masked, int lim, float slack) KVQ_INLINE {
    auto& t = s[decltype(par)::value];
    if (masked)
      each<0, 32>([&](auto e) KVQ_INLINE {
        constexpr int n = decltype(e)::value;
        t[n / 16][n % 16] = n < lim ? t[n / 16][n % 16] : -INFINITY;
      });
    float x = t[0][0];
    each<1, 32>([&](auto e) KVQ_INLINE { x = fmaxf(x, t[e.value / 16][e.value % 16]); });
    x = xmax32(x * kz);
    x = x > m + slack ? x : m;
    base = x == -INFINITY ? 0.0f : x;
    const float f = __builtin_amdgcn_exp2f(m - base);
    m = x;
    grow *= f;
    l *= f;
  };
  auto begin = [&]() KVQ_INLINE {
    safe = base - (kLift + lr);
    sum = 0.0f;
  };
  auto share = [&](auto par, auto which, auto again) KVQ_INLINE {
    // a pair's exponentials, then the pair before it: no wait for a result
    constexpr int i = decltype(which)::value, k = 2 * i;
    auto& t = s[decltype(par)::value];
    auto finish = [&](auto at) KVQ_INLINE {
      constexpr int n = decltype(at)::value;
      uint32_t w = pack2<BF16>(wx, wz);
      asm volatile("" : "+v"(w));             // here, not behind a branch
      p[decltype(par)::value][n / 8][n % 8 / 2] = w;
      // Sums of the rounded weights: what a large one loses leaves the sum as well (error against 64 bits, of a float32 softmax's: bf16
      // 1.50 -> 1.31, fp16 1.38-1.46 -> 1.21-1.33; time 1.00-1.02, the largest case 1.01).  Subnormal fp16 ones count.
      if constexpr (BF16) {
        sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w), __builtin_bit_cast(bf16x2, 0x3f803f80u), sum, false);
      } else {
        float y = sum;
        asm("v_fma_mix_f32 %0, %1, 1.0, %0 op_sel_hi:[1,0,0]" : "+v"(y) : "v"(w));
        asm("v_fma_mix_f32 %0, %1, 1.0, %0 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "+v"(y) : "v"(w));
        sum = y;
      }
    };
    float x = __builtin_fmaf(t[k / 16][k % 16], kz, -safe), z = __builtin_fmaf(t[k / 16][k % 16 + 1], kz, -safe);
    if constexpr (decltype(again)::value) {   // not above the reference's: it is off by much where scores pass 2^24 (a NaN stays one)
      x = x > kLift + lr ? kLift + lr : x;
      z = z > kLift + lr ? kLift + lr : z;
    }
    x = __builtin_amdgcn_exp2f(x);
    z = __builtin_amdgcn_exp2f(z);
    if constexpr (i > 0) finish(std::integral_constant<int, k - 2>{});
    wx = x;
    wz = z;
    if constexpr (i == 15) finish(std::integral_constant<int, k>{});
  };
  // The sum without the value scale, where that is so far below the unit that the type does not hold a weight times it: such weights may
  // be lost in the products, where they are nothing beside the larger block's, but not in the sum
  auto plain_sum = [&](auto par, auto again) KVQ_INLINE {
    float y = 0.0f;
    each<0, 32>([&](auto e) KVQ_INLINE {
      float x = __builtin_fmaf(s[decltype(par)::value][e.value / 16][e.value % 16], kz, kLift - base);
      if constexpr (decltype(again)::value) x = x > kLift ? kLift : x;
      y += __builtin_amdgcn_exp2f(x);
    });
    return y;
  };
  constexpr int kV = 4 * (D / 32), kK = 2 * (D / 16);               // steps of the two products
  constexpr std::integral_constant<int, 0> even{};
  constexpr std::integral_constant<int, 1> odd{};
  constexpr std::false_type no{};
  constexpr std::true_type yes{};
  auto add_v = [&](auto par, auto t, const u32x4& w) KVQ_INLINE {   // o += V P, operand t
    constexpr int c = decltype(t)::value % (D / 32), y = decltype(t)::value / (D / 32);
    o[c] = mfma32<BF16>(w, p[decltype(par)::value][y], o[c]);
  };
  // o += V P of the other parity (if `with`) beside the softmax of this one
  auto values = [&](auto par, bool look, bool masked, auto with, int lim) KVQ_INLINE {
    constexpr bool kWith = decltype(with)::value;
    constexpr std::integral_constant<int, 1 - decltype(par)::value> other{};
    u32x4 w[3];
    grow = 1.0f;
    if (look) find(par, masked, lim, 8.0f);
    begin();
    if constexpr (kWith) {
      w[0] = read_v(other, 0);
      w[1] = read_v(other, 1);
    }
    each<0, kV>([&](auto t) KVQ_INLINE {
      if constexpr (kWith) {
        if constexpr (t.value + 2 < kV) w[(t.value + 2) % 3] = read_v(other, t.value + 2);
        add_v(other, t, w[t.value % 3]);
      }
      each<t.value * 16 / kV, (t.value + 1) * 16 / kV>([&](auto i) KVQ_INLINE { share(par, i, no); });
      __builtin_amdgcn_sched_barrier(0);
    });
    float add = sum * inv_r;
    constexpr bool kFar = BF16 || !kOne;
    const bool far = kFar && inv_r > 2.0f / kWindow;
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(add > kMost || far) != 0, 0)) {
      if constexpr (kFar) add = far ? plain_sum(par, no) : add;
      if (__builtin_amdgcn_ballot_w64(add > kMost)) {
        find(par, false, lim, 0.0f);
        begin();
        each<0, 16>([&](auto i) KVQ_INLINE { share(par, i, yes); });
        add = sum * inv_r;
        if constexpr (kFar) add = far ? plain_sum(par, yes) : add;
      }
    }
    l += add;
    asm volatile("" : "+v"(l));
  };
  // S = K Q of the units of the other parity, beside `job` of each of its steps
  auto products = [&](auto par, auto&& job) KVQ_INLINE {
    constexpr int next = 1 - decltype(par)::value;
    constexpr std::integral_constant<int, next> other{};
    u32x4 w[4];
    each<0, 16>([&](auto e) KVQ_INLINE { s[next][0][e.value] = s[next][1][e.value] = 0.0f; });
    each<0, 3>([&](auto t) KVQ_INLINE { w[t.value] = read_k(other, t.value); });
    each<0, kK>([&](auto t) KVQ_INLINE {
      if constexpr (t.value + 3 < kK) w[(t.value + 3) % 4] = read_k(other, t.value + 3);
      s[next][t.value % 2] = mfma32<BF16>(w[t.value % 4], q[t.value / 2], s[next][t.value % 2]);
      job(t);
    });
  };
  auto nothing = [](auto) {};
  auto rescale = [&]() KVQ_INLINE {
    if (__builtin_amdgcn_ballot_w64(grow != 1.0f)) each<0, D / 32>([&](auto c) KVQ_INLINE { o[c.value] *= grow; });
  };
  // kz, lr and inv_r of a unit from its scales; what o is to be scaled by for a new unit of its own, which is each row's: only the
  // blocks that a row sees count (a hidden one may have any scale, NaN too; far larger ones behind a row cost it its fp16 weights).  bf16
  // blocks have scales down to 2^-109, with codes down to 2^-108; in fp16 what is below 2^-100 is a block of zeros, which weighs nothing in o.
  float turn = 1.0f;
  auto above = [](float x) KVQ_INLINE { return __uint_as_float((__float_as_uint(x) & 0x7f800000u) + 0x00800000u); };  // the next 2^k
  auto scale_for = [&](float2 z, bool masked, int lim) KVQ_INLINE {
    kz = z.x * a.scale;
    kz = kz < FLT_MIN ? FLT_MIN : kz;
    turn = 1.0f;
    float v = z.y;
    if (masked) v = (kOne ? lim + 32 * g : lim) > 0 ? v : 0.0f;
    if constexpr (!kOne) v = xmax32(v);
    // changed where a scale is not within the window below it (fp16: its weights have to stay normal numbers; bf16: their sum)
    constexpr float kEmpty = BF16 ? 0.0f : 0x1p-100f;
    const bool out = v != __builtin_amdgcn_fmed3f(v, unit * kWindow, unit);
    if (__builtin_amdgcn_ballot_w64(out)) {
      const bool change = out && v > kEmpty;   // not for a NaN, or where the row sees nothing
      float now = above(v);
      if (__builtin_amdgcn_ballot_w64(change && now < unit)) {
        // a fall multiplies o: not beyond 2^122, the products that are on their way to it (below 2^32) with it
        float most = 0x1p32f;
        each<0, D / 32>([&](auto c) KVQ_INLINE { each<0, 16>([&](auto e) KVQ_INLINE { most = fmaxf(most, fabsf(o[c.value][e.value])); }); });
        const float least = unit * (above(fminf(xmax32(most), 0x1p120f)) * 0x1p-121f);
        now = now < least ? least : now;
      }
      turn = change && unit > 0.0f ? unit / now : 1.0f;
      unit = change ? now : unit;
    }
    // (the quotient of a power of two is exact; a scale is taken for 2^-100 of its unit at least)
    float r = z.y < kEmpty ? 1.0f : z.y * __builtin_amdgcn_rcpf(unit);
    r = r < 0x1p-100f ? 0x1p-100f : r;
    lr = __builtin_amdgcn_logf(r);
    inv_r = __builtin_amdgcn_rcpf(r);
    if (masked) {
      kz = lim > 0 ? kz : 1.0f;
      lr = lim > 0 ? lr : 0.0f;
      inv_r = lim > 0 ? inv_r : 0.0f;
    }
  };
  // (nothing of what lies behind the last unit, for either half)
  auto lim_of = [&](int j) KVQ_INLINE { return j < units ? (visible < full ? visible : full) - (u0 + j) * kUnit - 32 * g : -kUnit; };
  // Pages of units on their way: id[i] of unit j + 1 + i when iteration j begins
  Ids id[3], next_id;
  float2 z_now;
  auto step = [&](auto par, int j) KVQ_INLINE {
    constexpr int kPar = decltype(par)::value;
    const bool masked = j >= whole;
    const int lim = lim_of(j);
    scale_for(z_now, masked, lim);
    z_now = scales_of(id[0]);
    next_id = ids_of(j + 4);
    __builtin_amdgcn_s_setprio(1);            // the softmax goes before the other wavefront's products
    values(par, masked, true, yes, lim);
    __builtin_amdgcn_s_setprio(0);
    grow *= turn;
    // unit j + 2 of K and j of V into the buffers of this parity, then the codes of the ones after them
    products(par, [&](auto t) KVQ_INLINE {
      constexpr int kJobs = 4 * kPer, kFirst = t.value * kJobs / kK, kEnd = (t.value + 1) * kJobs / kK;
      each<kFirst, kEnd>([&](auto i) KVQ_INLINE {
        if constexpr (i.value < 2 * kPer) {
          widen_k(kPar, i);
          if constexpr (i.value % 2) fetch_k(id[2], j + 3, std::integral_constant<int, i.value / 2>{});
        } else {
          constexpr std::integral_constant<int, i.value - 2 * kPer> v{};
          widen_v(kPar, v);
          if constexpr (v.value % 2) fetch_v(id[0], j + 1, std::integral_constant<int, v.value / 2>{});
        }
      });
    });
    rescale();
    id[0] = id[1];
    id[1] = id[2];
    id[2] = next_id;
    block_lds_barrier();
  };
  each<0, D / 16>([&](auto i) { q[i.value] = (q[i.value] ^ a.sign) & mask; });
  if (tiles) {
    const Ids first = ids_of(0);
    id[0] = ids_of(1);
    id[1] = ids_of(2);
    id[2] = ids_of(3);
    // keys of two units and values of one on their way at once
    each<0, kPer>([&](auto i) { fetch_k(id[0], 1, i); });
    u32x4 later[kPer];
    each<0, kPer>([&](auto i) { later[i.value] = kw[i.value]; });
    each<0, kPer>([&](auto i) { fetch_k(first, 0, i); });
    each<0, kPer>([&](auto i) { fetch_v(first, 0, i); });
    z_now = scales_of(first);
    each<0, 2 * kPer>([&](auto i) { widen_k(0, i); });
    each<0, kPer>([&](auto i) { kw[i.value] = later[i.value]; });
    each<0, 2 * kPer>([&](auto i) { widen_k(1, i); });
    each<0, kPer>([&](auto i) { fetch_k(id[1], 2, i); });
    each<0, 2 * kPer>([&](auto i) { widen_v(0, i); });
    each<0, kPer>([&](auto i) { fetch_v(id[0], 1, i); });
    block_lds_barrier();
    products(odd, nothing);                   // unit 0
    const int lim = lim_of(0);
    scale_for(z_now, whole == 0, lim);
    z_now = scales_of(id[0]);
    if (tiles > 1) {
      block_lds_barrier();                    // K(2) takes the place of K(0)
      each<0, 2 * kPer>([&](auto i) { widen_k(0, i); });
      each<0, kPer>([&](auto i) { fetch_k(id[2], 3, i); });
    }
    values(even, true, whole == 0, no, lim);
    if (__builtin_amdgcn_ballot_w64(live && m == -INFINITY)) whole = 0;      // a row without a reference yet
    if (tiles > 1) {
      products(even, nothing);                // unit 1
      // ids of units 2, 3, 4
      id[0] = id[1];
      id[1] = id[2];
      id[2] = ids_of(4);
      block_lds_barrier();
    }
    for (int j = 1; j < tiles; j += 2) {
      step(odd, j);
      step(even, j + 1);
    }
    each<0, kV>([&](auto t) KVQ_INLINE { add_v(even, t, read_v(even, t.value)); });
  }
  each<0, D / 32>([&](auto c) KVQ_INLINE { o[c.value] *= unit; });

  // Units of the open block
  const int64_t open = ((static_cast<int64_t>(slot) * 2 + buf) * a.H + h) * P * D;
  const uint16_t *ko = a.ko + open, *vo = a.vo + open;
  const int first_open = u0 > u_full ? u0 : u_full;
  for (int u = first_open; u < u1; ++u) {
    const int off = (u - u_full) * kUnit, t0 = full + off, rest = len - t0 < kUnit ? len - t0 : kUnit;
    constexpr int kMine = kUnit * kPieces / kThreads;
    u32x4 kx[kMine], vx[kMine];               // behind the last token: zeros
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int x = tid + i * kThreads, t = x / kPieces, ch = x / 8;
      kx[i] = vx[i] = u32x4{0, 0, 0, 0};
      if (t < rest) kx[i] = *reinterpret_cast<const u32x4*>(ko + (off + t) * D + 8 * (x % kPieces));
      if (8 * (x % 8) < rest) vx[i] = *reinterpret_cast<const u32x4*>(vo + ch * P + off + 8 * (x % 8));
    }
    __syncthreads();
    // what is hidden from a row may be an infinity or a NaN, and what lies behind the last token anything: such values go in as
    // zeros, and the rows that do see one have it afterwards
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int x = tid + i * kThreads;
      k_put(0, x / kPieces, x % kPieces, kx[i]);
      u32x4 w = vx[i];
      bool bad = false;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool i0 = (w[e] & kInf) == kInf, i1 = (w[e] >> 16 & kInf) == kInf;
        bad |= i0 || i1;
        w[e] = (i0 ? 0u : w[e] & 0xffffu) | (i1 ? 0u : w[e] & 0xffff0000u);
      }
      v_put(0, x / 8, x % 8, w);
      if (bad) flag[u - u_full] = 1;
    }
    __syncthreads();
    products(odd, nothing);
    kz = a.scale;
    lr = 0.0f;
    inv_r = 1.0f;
    values(even, true, true, no, visible - t0 - 32 * g);
    rescale();
    each<0, kV>([&](auto t) KVQ_INLINE { add_v(even, t, read_v(even, t.value)); });
  }
  // A visible value that is infinite or NaN is its channel's result, however small its weight
  for (int u = first_open; u < u1; ++u) {
    const int off = (u - u_full) * kUnit, t0 = full + off, rest = len - t0 < kUnit ? len - t0 : kUnit;
    if (!flag[u - u_full]) continue;
    for (int t = 0; t < rest; ++t)
      each<0, D / 32>([&](auto c) {
        each<0, 16>([&](auto e) {
          const uint16_t x = vo[(32 * c.value + 8 * (e.value / 4) + 4 * g + e.value % 4) * P + off + t];
          if (t0 + t < visible && (x & kInf) == kInf) o[c.value][e.value] += BF16 ? bf16_to_f32(x) : f16_to_f32(x);
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

// D / 4 lanes per row that is joined of several parts, its sums 16 bytes a lane: those of its own tile and those of a tile of its
// shared front, four on their way at once.  SPREAD: a workgroup per row, for many parts of few rows.  What bounds it: the parts'
// way from memory (16 questions of 17 to 391 tokens behind 8131, 123 MB of them: 19-21 us, 6 TB/s).
template <int D, bool BF16, int W, bool SPREAD>
__global__ __launch_bounds__(kThreads) void paged_wide_merge_kernel(WideArgs a, const int* __restrict__ merges) {
  constexpr int kTileRows = 32 * W, kLanes = D / 4, kGroups = kThreads / kLanes;
  const int* w = merges + kMergeWords * (blockIdx.x / a.H);
  const int group = threadIdx.x / kLanes, h = blockIdx.x % a.H, lane = threadIdx.x % kLanes, row = SPREAD ? blockIdx.y : blockIdx.y * kGroups + group;
  const int tok = row / a.rep, hq = row % a.rep;
  if (tok >= w[1]) return;
  constexpr int64_t kPart = kTileRows * (D + 2);
  const int64_t stride = a.H * kPart;
  float top = -INFINITY, l = 0.0f;
  f32x4 o = {0, 0, 0, 0};
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const int first = w[2 + 3 * side], parts = w[3 + 3 * side], r = (w[4 + 3 * side] + tok) * a.rep + hq;
    const int from = SPREAD ? parts * group / kGroups : 0, to = SPREAD ? parts * (group + 1) / kGroups : parts;
    const float* part = a.part + (static_cast<int64_t>(first) * a.H + h) * kPart;
    for (int i0 = from; i0 < to; i0 += 4) {   // behind the last: it again, unused
      f32x4 x[4];
      float2 st[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float* at = part + (i0 + k < to ? i0 + k : to - 1) * stride;
        x[k] = *reinterpret_cast<const f32x4*>(at + r * D + 4 * lane);
        st[k] = *reinterpret_cast<const float2*>(at + kTileRows * D + 2 * r);
      }
      float m = top;
#pragma unroll
      for (int k = 0; k < 4; ++k) m = fmaxf(m, st[k].x);
      const float safe = m == -INFINITY ? 0.0f : m, old = __builtin_amdgcn_exp2f(top - safe);
      top = m;
      l *= old;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = weigh(old, o[e]);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (i0 + k >= to) break;
        const float f = __builtin_amdgcn_exp2f(st[k].x - safe);
        l += f * st[k].y;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] += weigh(f, x[k][e]);
      }
    }
  }
  if constexpr (SPREAD) {
    __shared__ f32x4 sums[kGroups][kLanes];
    __shared__ float2 stats[kGroups];
    sums[group][lane] = o;
    if (lane == 0) stats[group] = make_float2(top, l);
    __syncthreads();                          // a workgroup is one row: all or none get here
    if (group) return;
    top = stats[0].x;
#pragma unroll
    for (int k = 1; k < kGroups; ++k) top = fmaxf(top, stats[k].x);
    const float safe = top == -INFINITY ? 0.0f : top;
    l = 0.0f;
    o = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < kGroups; ++k) {
      const float f = __builtin_amdgcn_exp2f(stats[k].x - safe);
      l += f * stats[k].y;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += weigh(f, sums[k][lane][e]);
    }
  }
  const float inv = 1.0f / l;                 // a row that is joined sees a token at least
  uint16_t* out = a.out + ((w[0] + static_cast<int64_t>(tok)) * a.H * a.rep + h * a.rep + hq) * D + 4 * lane;
  *reinterpret_cast<uint2*>(out) = make_uint2(pack2<BF16>(o[0] * inv, o[1] * inv), pack2<BF16>(o[2] * inv, o[3] * inv));
}

template <int D>
void launch_wide(const WideArgs& a, int page, int code, bool bf16, int waves, int64_t items, int64_t merges, int64_t most_parts, hipStream_t stream) {
  auto run = [&](auto p, auto c, auto t, auto w) {
    constexpr int P_ = decltype(p)::value, C_ = decltype(c)::value, W_ = decltype(w)::value;
    constexpr bool T_ = decltype(t)::value;
    hipLaunchKernelGGL((paged_wide_kernel<D, P_, C_, T_, W_>), dim3(static_cast<uint32_t>(items * a.H)), dim3(64 * W_), 0, stream, a);
    const uint32_t x = static_cast<uint32_t>(merges * a.H);
    const int* words = a.items + kItemWords * items;
    if (merges && most_parts >= kSpread)
      hipLaunchKernelGGL((paged_wide_merge_kernel<D, T_, W_, true>), dim3(x, 32 * W_), dim3(kThreads), 0, stream, a, words);
    else if (merges)
      hipLaunchKernelGGL((paged_wide_merge_kernel<D, T_, W_, false>), dim3(x, 32 * W_ * (D / 4) / kThreads), dim3(kThreads), 0, stream, a, words);
  };
  auto by_waves = [&](auto p, auto c, auto t) {
    if constexpr (D == 128) {
      if (waves == 8) return run(p, c, t, std::integral_constant<int, 8>{});
    }
    run(p, c, t, std::integral_constant<int, 4>{});
  };
  auto by_type = [&](auto p, auto c) {
    if (bf16) by_waves(p, c, std::true_type{});
    else by_waves(p, c, std::false_type{});
  };
  auto by_code = [&](auto p) {
    if (code == kCodeInt8) by_type(p, std::integral_constant<int, kCodeInt8>{});
    else by_type(p, std::integral_constant<int, kCodeE4M3>{});
  };
  if (page == 32) by_code(std::integral_constant<int, 32>{});
  else if (page == 64) by_code(std::integral_constant<int, 64>{});
  else by_code(std::integral_constant<int, 128>{});
}

}  // namespace
}  // namespace kvq
